// tq_rope.cu — norm and rotation of query and key heads in one pass
// (tq_qk_rope): y = rotation(x / rms(x) * w) in fp32, rounded once.
//
// Bound by HBM: a head vector is read and written once, a token's row of the
// rotation table once for its heads.  rope_rows_kernel: LV lanes hold a
// vector in registers, 8 (16-bit) or 4 (32-bit) of its values in each of two
// 16-byte pieces that hold each other's rotation partners (dims i and rot/2 +
// i, or neighbours when interleaved), so the rotation needs no exchange and
// only the norm's sum crosses lanes.  A group of lanes takes kHeads heads of
// one token, all their loads in flight, with the token's cosines and sines
// (times the weights) in registers, and works on fp32 pairs: with scalar
// arithmetic the instructions, not HBM, set the time.  Views that do not take
// 16-byte accesses (and heads of odd sizes or rotary parts) run rope_any_kernel,
// a warp per vector.
// 16,381 tokens x 48 heads of 128, bf16, normed: 89.5 us for 411 MB, 4.6 TB/s (a
// plain copy of the bytes takes 64); 16 tokens 4.1 us, the launch.  The 16-bit
// instances spill 40-48 bytes a thread at the 80 registers of three CTAs an SM; two
// CTAs of 126 registers without a spill took 97 us.
#include "tq_internal.h"
#include "tq_ragged.cuh"
#include "tq_tc.cuh"

namespace tq {
namespace {

struct RopeSide {
  const void* x;
  void* y;
  int64_t xs[4], ys[4];
  int64_t H;
  int dtype;
  HeadXform f;
};

struct RopeParams {
  RopeSide side[2];             // q, k (H = 0: absent)
  int64_t B, T;
  int D;
  const void* pos; int pos64; int64_t ps[2];
  uint32_t* status;
};

constexpr int kRopeWarps = 8;

__device__ __forceinline__ int64_t load_pos(const void* pos, int pos64, int64_t i) {
  return pos64 ? __ldg(reinterpret_cast<const long long*>(pos) + i)
               : (int64_t)__ldg(reinterpret_cast<const int*>(pos) + i);
}

// Any type, stride, head size and rotary part: one warp per head vector, the
// vector staged in shared memory.
__global__ void __launch_bounds__(32 * kRopeWarps) rope_any_kernel(RopeParams p) {
  __shared__ float rows[kRopeWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* u = rows[warp];
  const int64_t Hs = p.side[0].H + p.side[1].H, total = p.B * p.T * Hs;
  for (int64_t i = blockIdx.x * (int64_t)kRopeWarps + warp; i < total;
       i += (int64_t)gridDim.x * kRopeWarps) {
    const int64_t tok = i / Hs, b = tok / p.T, t = tok % p.T;
    int64_t h = i % Hs;
    const int w = h >= p.side[0].H;
    if (w) h -= p.side[0].H;
    const RopeSide& s = p.side[w];
    const int64_t xb = b * s.xs[0] + h * s.xs[1] + t * s.xs[2];
    for (int c = lane; c < p.D; c += 32) u[c] = load_elem(s.x, s.dtype, xb + c * s.xs[3]);
    __syncwarp();
    int64_t row = 0;
    if (s.f.cos_sin)
      row = table_row(s.f, load_pos(p.pos, p.pos64, b * p.ps[0] + t * p.ps[1]), p.status);
    xform_row(u, p.D, s.f, row, lane);
    const int64_t yb = b * s.ys[0] + h * s.ys[1] + t * s.ys[2];
    for (int c = lane; c < p.D; c += 32) store_elem(s.y, s.dtype, yb + c * s.ys[3], u[c]);
    __syncwarp();
  }
}

// Heads of a token per group of lanes: 16,381 tokens 89 us, with 2 heads 103 (the
// table is read more often), with 8 98 (registers: fewer CTAs).
constexpr int kHeads = 4;
constexpr int kRowThreads = 256;

using tc::f2;

// P values of a piece, as fp32 pairs and back.
template <int DT>
struct Piece {
  static constexpr int ES = DT == TQ_F32 ? 4 : 2, P = 16 / ES;
  uint4 raw;
  __device__ __forceinline__ void load(const void* x, int64_t i) {
    // a plain load: the output may be the input
    raw = *reinterpret_cast<const uint4*>(static_cast<const char*>(x) + i * ES);
  }
  __device__ __forceinline__ void widen(f2 (&v)[P / 2]) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (ES == 4) {
      v[0] = tc::f2_make(__uint_as_float(w[0]), __uint_as_float(w[1]));
      v[1] = tc::f2_make(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == TQ_BF16) {
          v[i] = tc::f2_make(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[i] = tc::f2_make(f.x, f.y);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(void* y, int64_t i, const f2 (&v)[P / 2]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < P / 2; ++k) {
      float lo, hi;
      tc::f2_split(v[k], lo, hi);
      if constexpr (ES == 4) {
        w[2 * k] = __float_as_uint(lo);
        w[2 * k + 1] = __float_as_uint(hi);
      } else if constexpr (DT == TQ_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        w[k] = pack_half2(lo, hi);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<char*>(y) + i * ES) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// n consecutive fp32 values, 16-byte aligned.
template <int N>
__device__ __forceinline__ void load_f32(float (&v)[N], const float* p) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
    v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
  }
}

// P weights from dim d on, plus the offset.
template <int P>
__device__ __forceinline__ void load_weights(float (&w)[P], const HeadXform& f, int d) {
  const int bytes = f.w_dtype == TQ_F32 ? 4 * P : 2 * P;
  const char* at = static_cast<const char*>(f.weight) + (int64_t)d * (bytes / P);
  if ((reinterpret_cast<uintptr_t>(f.weight) & 15) == 0) {  // pieces of 8, 16 or 32 bytes
    if (f.w_dtype == TQ_F32) {
      load_f32<P>(w, reinterpret_cast<const float*>(at));
    } else {
#pragma unroll
      for (int i = 0; i < P; i += 4) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(at + 2 * i));
        const uint32_t h[2] = {u.x, u.y};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 x = f.w_dtype == TQ_F16
                               ? __half22float2(*reinterpret_cast<const __half2*>(&h[k]))
                               : make_float2(__uint_as_float(h[k] << 16),
                                             __uint_as_float(h[k] & 0xFFFF0000u));
          w[i + 2 * k] = x.x;
          w[i + 2 * k + 1] = x.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < P; ++e) w[e] = load_elem(f.weight, f.w_dtype, d + e);
  }
#pragma unroll
  for (int e = 0; e < P; ++e) w[e] += f.w_offset;
}

// D = 2 P LV values per vector.  Groups of LV lanes; a group's unit is (token,
// run of kHeads heads of q or k).
template <int DT, int LV, bool PAIRS>
__global__ void __launch_bounds__(kRowThreads, 3) rope_rows_kernel(RopeParams p, int runs_q, int runs) {
  using X = Piece<DT>;
  constexpr int P = X::P, D = 2 * P * LV;
  const int l = threadIdx.x % LV;
  const uint32_t unit = blockIdx.x * (uint32_t)(kRowThreads / LV) + threadIdx.x / LV;
  const uint32_t tok = unit / (uint32_t)runs;
  if (tok >= (uint32_t)(p.B * p.T)) return;                // whole groups leave together
  const int run = (int)(unit - tok * (uint32_t)runs), w = run >= runs_q;
  const RopeSide& s = p.side[w];
  const int h0 = (w ? run - runs_q : run) * kHeads;
  const int nh = tmin(kHeads, (int)s.H - h0);
  const uint32_t b = tok / (uint32_t)p.T, t = tok - b * (uint32_t)p.T;
  // the two pieces: rotation partners, or halves of the vector
  const int half = s.f.rot / 2;
  int ga = P * l, gb = D / 2 + P * l;
  bool turn_a = s.f.cos_sin != nullptr, turn_b = turn_a;
  if (PAIRS) {
    turn_b = false;
    if (ga < half) { gb = half + ga; }
    else { ga = s.f.rot + 2 * (P * l - half); gb = ga + P; turn_a = false; }
  } else {
    turn_a = turn_a && ga < s.f.rot;
    turn_b = turn_b && gb < s.f.rot;
  }
  const int64_t xb = b * s.xs[0] + t * s.xs[2] + (int64_t)h0 * s.xs[1];
  X a[kHeads], c[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    a[i].raw = c[i].raw = make_uint4(0u, 0u, 0u, 0u);
    if (i < nh) {
      a[i].load(s.x, xb + i * s.xs[1] + ga);
      c[i].load(s.x, xb + i * s.xs[1] + gb);
    }
  }
  // The token's coefficients, weights folded in: piece a becomes u A + v B, piece
  // b becomes v C + u E (pairs), or u A + swap(u) B and v C + swap(v) E with
  // swap exchanging the neighbours of a pair (interleaved).
  f2 A[P / 2], B[P / 2], C[P / 2], E[P / 2];
  {
    float wa[P], wb[P], cs[P], sn[P];
#pragma unroll
    for (int e = 0; e < P; ++e) wa[e] = wb[e] = 1.f;
    if (s.f.weight) {
      load_weights<P>(wa, s.f, ga);
      load_weights<P>(wb, s.f, gb);
    }
    const float* tab = s.f.cos_sin;
    if (tab)
      tab += table_row(s.f, load_pos(p.pos, p.pos64, b * p.ps[0] + t * p.ps[1]), p.status) * s.f.rot;
    if (PAIRS) {
      if (turn_a) { load_f32<P>(cs, tab + ga); load_f32<P>(sn, tab + half + ga); }
#pragma unroll
      for (int e = 0; e < P; e += 2) {
        const float c0 = turn_a ? cs[e] : 1.f, c1 = turn_a ? cs[e + 1] : 1.f;
        const float s0 = turn_a ? sn[e] : 0.f, s1 = turn_a ? sn[e + 1] : 0.f;
        A[e / 2] = tc::f2_make(wa[e] * c0, wa[e + 1] * c1);
        B[e / 2] = tc::f2_make(-wb[e] * s0, -wb[e + 1] * s1);
        C[e / 2] = tc::f2_make(wb[e] * c0, wb[e + 1] * c1);
        E[e / 2] = tc::f2_make(wa[e] * s0, wa[e + 1] * s1);
      }
    } else {
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        const float ca = turn_a ? __ldg(tab + ga / 2 + i) : 1.f;
        const float sa = turn_a ? __ldg(tab + half + ga / 2 + i) : 0.f;
        const float cb = turn_b ? __ldg(tab + gb / 2 + i) : 1.f;
        const float sb = turn_b ? __ldg(tab + half + gb / 2 + i) : 0.f;
        A[i] = tc::f2_make(wa[2 * i] * ca, wa[2 * i + 1] * ca);
        B[i] = tc::f2_make(-wa[2 * i + 1] * sa, wa[2 * i] * sa);
        C[i] = tc::f2_make(wb[2 * i] * cb, wb[2 * i + 1] * cb);
        E[i] = tc::f2_make(-wb[2 * i + 1] * sb, wb[2 * i] * sb);
      }
    }
  }
  const int64_t yb = b * s.ys[0] + t * s.ys[2] + (int64_t)h0 * s.ys[1];
  // The sums cross lanes, and a warp holds groups of q and of k, so every lane
  // takes part where either side has a norm, and heads past a run's end are
  // worked on too (zeros).
  const bool normed = p.side[0].f.weight != nullptr || p.side[1].f.weight != nullptr;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    f2 u[P / 2], v[P / 2];
    a[i].widen(u);
    c[i].widen(v);
    if (normed) {
      f2 sq = tc::f2_mul(u[0], u[0]);
      sq = tc::f2_fma(v[0], v[0], sq);
#pragma unroll
      for (int e = 1; e < P / 2; ++e) sq = tc::f2_fma(v[e], v[e], tc::f2_fma(u[e], u[e], sq));
      float lo, hi;
      tc::f2_split(sq, lo, hi);
      float ss = lo + hi;
#pragma unroll
      for (int o = LV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = s.f.weight ? rsqrtf(fmaf(ss, 1.f / (float)D, s.f.eps)) : 1.f;
      const f2 rr = tc::f2_make(r, r);
#pragma unroll
      for (int e = 0; e < P / 2; ++e) {
        u[e] = tc::f2_mul(u[e], rr);
        v[e] = tc::f2_mul(v[e], rr);
      }
    }
    f2 y[P / 2], z[P / 2];
    auto swap = [](f2 x) {
      float lo, hi;
      tc::f2_split(x, lo, hi);
      return tc::f2_make(hi, lo);
    };
    // dims that are not rotated take no other's value, not even times zero
#pragma unroll
    for (int e = 0; e < P / 2; ++e) {
      y[e] = tc::f2_mul(u[e], A[e]);
      z[e] = tc::f2_mul(v[e], C[e]);
      if (turn_a) y[e] = tc::f2_fma(PAIRS ? v[e] : swap(u[e]), B[e], y[e]);
      if (PAIRS ? turn_a : turn_b) z[e] = tc::f2_fma(PAIRS ? u[e] : swap(v[e]), E[e], z[e]);
    }
    if (i < nh) {
      X::store(s.y, yb + i * s.ys[1] + ga, y);
      X::store(s.y, yb + i * s.ys[1] + gb, z);
    }
  }
}

// 16-byte accesses: unit last stride, every other stride and the base aligned.
bool takes_pieces(const tq_tensor4* x) {
  const int es = x->dtype == TQ_F32 ? 4 : 2;
  if (x->stride[3] != 1 || reinterpret_cast<uintptr_t>(x->data) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (x->shape[i] > 1 && (x->stride[i] * es) % 16) return false;
  return true;
}

using RopeFn = void (*)(RopeParams, int, int);

template <int DT, bool PAIRS>
RopeFn rows_fn(int lanes) {
  switch (lanes) {
    case 2: return rope_rows_kernel<DT, 2, PAIRS>;
    case 4: return rope_rows_kernel<DT, 4, PAIRS>;
    case 8: return rope_rows_kernel<DT, 8, PAIRS>;
    case 16: return rope_rows_kernel<DT, 16, PAIRS>;
    case 32: return rope_rows_kernel<DT, 32, PAIRS>;
    default: return nullptr;
  }
}

}  // namespace

int launch_qk_rope(const tq_rope* rope, const tq_positions* pos, const tq_tensor4* const x[2],
                   const tq_tensor4* const y[2], const tq_head_norm* const norm[2],
                   uint32_t* status, cudaStream_t st) {
  RopeParams p = {};
  for (int w = 0; w < 2; ++w) {
    RopeSide& s = p.side[w];
    s.H = 0;
    if (!x[w]) continue;
    s.x = x[w]->data; s.y = y[w]->data; s.dtype = x[w]->dtype;
    for (int i = 0; i < 4; ++i) { s.xs[i] = x[w]->stride[i]; s.ys[i] = y[w]->stride[i]; }
    s.H = x[w]->shape[1];
    s.f = head_xform(rope, norm[w]);
    p.B = x[w]->shape[0];
    p.T = x[w]->shape[2];
    p.D = (int)x[w]->shape[3];
  }
  p.pos = pos ? pos->data : nullptr;
  p.pos64 = pos && pos->bits == 64;
  p.ps[0] = pos ? pos->stride[0] : 0;
  p.ps[1] = pos ? pos->stride[1] : 0;
  p.status = status;
  const int64_t total = p.B * p.T * (p.side[0].H + p.side[1].H);
  if (total == 0) return TQ_OK;
  // the register kernel: both sides of one type and 16-byte accesses, D / 2
  // pieces over 2..32 lanes, a rotary part of whole pieces
  const tq_tensor4* one = x[0] ? x[0] : x[1];
  const int es = one->dtype == TQ_F32 ? 4 : 2, P = 16 / es;
  bool rows = p.D % (2 * P) == 0 && (!rope || rope->rot_dim % (2 * P) == 0);
  for (int w = 0; w < 2; ++w)
    if (x[w])
      rows = rows && x[w]->dtype == one->dtype && takes_pieces(x[w]) && takes_pieces(y[w]);
  const bool halves = rope && !rope->interleaved;
  RopeFn fn = nullptr;
  if (rows) {
    const int lanes = p.D / (2 * P);
    fn = one->dtype == TQ_F32   ? (halves ? rows_fn<TQ_F32, true>(lanes) : rows_fn<TQ_F32, false>(lanes))
         : one->dtype == TQ_F16 ? (halves ? rows_fn<TQ_F16, true>(lanes) : rows_fn<TQ_F16, false>(lanes))
                                : (halves ? rows_fn<TQ_BF16, true>(lanes) : rows_fn<TQ_BF16, false>(lanes));
  }
  if (fn) {
    const int lanes = p.D / (2 * P), per = kRowThreads / lanes;
    const int runs_q = (int)((p.side[0].H + kHeads - 1) / kHeads);
    const int runs = runs_q + (int)((p.side[1].H + kHeads - 1) / kHeads);
    const int64_t units = p.B * p.T * runs;
    if (units <= INT32_MAX - kRowThreads) {
      fn<<<(unsigned)((units + per - 1) / per), kRowThreads, 0, st>>>(p, runs_q, runs);
      return check_launch("tq_qk_rope");
    }
  }
  const int64_t blocks = (total + kRopeWarps - 1) / kRopeWarps;
  rope_any_kernel<<<(unsigned)tmin<int64_t>(blocks, 16 * device_sm_count()), 32 * kRopeWarps, 0,
                    st>>>(p);
  return check_launch("tq_qk_rope");
}

}  // namespace tq
