// tq_norm.cu — a block's output onto the residual stream, and the next block's
// norm of the sum (tq_residual_norm), a row at a time:
//   z = post(x),  y = residual + scale act(gate) z,  h = pre(y)
// with norms (x - mean) / sqrt(mean (x - mean)^2 + eps) (w + offset) + b, the
// mean taken off only where the norm is centred (layer norm; else RMS norm).
//
// Bound by HBM: x, residual and a gate of its own per element are read once, y and h
// written once; in fact by instructions beside it (issue slots 72 % busy).  16,381 rows
// of 4,096 (bf16, channel gate) 110 us for 537 MB, 4.9 TB/s; 16 rows of 5,120 4.6 us on
// the GPU; 2,051 rows of 2,050 (4-byte chunks, gate per element, layer norms) 35 us.  Sums go by
// shuffles and one barrier each, in an order that the width and the accesses that the views
// allow settle, so that a row called by itself is the row of a batch to the bit; h is formed
// from y before its rounding.
#include "tq_common.cuh"
#include "tq_internal.h"
#include "tq_tc.cuh"

#include <type_traits>

namespace tq {
namespace {

struct NormSide {
  int on, centered, dtype;
  const void* w;                // [C] or NULL: ones
  const void* b;                // [C] or NULL: zeros
  float eps, offset;
};

struct NormParams {
  const void* x; const void* r; const void* g;
  void* y; void* h;             // h: NULL without a norm behind the sum
  int gd;                       // gate's type
  int gmode;                    // 0: none, 1: a value per element, 2: one per row
  int act;
  float scale;
  int64_t xs[4], rs[4], gs[4], ys[4], hs[4];
  int64_t rows, n1, n2;         // rows: [rows / (n1 n2)][n1][n2], below 2^31; n2 = 0: one dim, stride [2]
  int C;
  NormSide post, pre;
};

// V consecutive values of type DT, as they lie in memory.
template <int DT, int V>
struct Chunk {
  static constexpr int ES = DT == TQ_F32 ? 4 : 2, B = ES * V;
  using Word = typename std::conditional<B == 2, uint16_t, uint32_t>::type;
  static constexpr int NW = B < 4 ? 1 : B / 4;
  Word w[NW];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    // plain loads: an output may be its input
    const char* at = static_cast<const char*>(base) + i * ES;
    if constexpr (B >= 16) {
#pragma unroll
      for (int k = 0; k < NW; k += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(at + 4 * k);
        w[k] = u.x; w[k + 1] = u.y; w[k + 2] = u.z; w[k + 3] = u.w;
      }
    } else if constexpr (B == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(at);
      w[0] = u.x; w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const Word*>(at);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < NW; ++k) w[k] = 0;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == TQ_F32) return __uint_as_float(w[e]);
    else {
      const uint32_t u = V == 1 ? (uint32_t)w[0] : (uint32_t)w[e / 2] >> (16 * (e & 1));
      if constexpr (DT == TQ_BF16) return __uint_as_float(u << 16);
      else return __half2float(__ushort_as_half((unsigned short)u));
    }
  }
  // values e, e + 1 (e even)
  __device__ __forceinline__ tc::f2 pair(int e) const {
    if constexpr (DT == TQ_F32) return tc::f2_make(__uint_as_float(w[e]), __uint_as_float(w[e + 1]));
    else if constexpr (DT == TQ_BF16)
      return tc::f2_make(__uint_as_float((uint32_t)w[e / 2] << 16), __uint_as_float(w[e / 2] & 0xFFFF0000u));
    else {
      const uint32_t u = w[e / 2];
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&u));
      return tc::f2_make(h.x, h.y);
    }
  }
  static __device__ __forceinline__ void store(void* base, int64_t i, const float* v) {
    char* at = static_cast<char*>(base) + i * ES;
    uint32_t o[NW];
    if constexpr (DT == TQ_F32) {
#pragma unroll
      for (int k = 0; k < NW; ++k) o[k] = __float_as_uint(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float lo = v[2 * k], hi = V == 1 ? 0.f : v[2 * k + (V > 1)];
        if constexpr (DT == TQ_BF16) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
          o[k] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          o[k] = pack_half2(lo, hi);
        }
      }
    }
    if constexpr (B >= 16) {
#pragma unroll
      for (int k = 0; k < NW; k += 4)
        *reinterpret_cast<uint4*>(at + 4 * k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
    } else if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(at) = make_uint2(o[0], o[1]);
    } else {
      *reinterpret_cast<Word*>(at) = (Word)o[0];
    }
  }
};

// V values of a parameter of any of the types (contiguous; V >= 2 aligned to V values).
template <int V>
__device__ __forceinline__ void load_param(float (&v)[V], const void* base, int dtype, int64_t i) {
  if (dtype == TQ_F32) {
    Chunk<TQ_F32, V> c;
    c.load(base, i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c.get(e);
  } else {
    Chunk<TQ_F16, V> c;
    c.load(base, i);
    if (dtype == TQ_F16) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = c.get(e);
    } else {
      Chunk<TQ_BF16, V> d;
#pragma unroll
      for (int k = 0; k < c.NW; ++k) d.w[k] = c.w[k];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = d.get(e);
    }
  }
}

// 1 / (1 + e^-g): e^-g = 2^t (1 + d ln 2) with t + d = -g log2 e in two parts, as t alone is
// off by |g| 2^-24 (the library's exponential and quotient took half of the instructions of a
// gated row).  Off by 2^-21 + 2^-22 at most: the exponential's 2^-22, four roundings, the
// quotient's 2 ulp (the worst of 4 million gates from -87 to 87: 5.0 x 2^-24); below 2^-126 it is 0.
__device__ __forceinline__ float activate(float g, int act) {
  if (act == TQ_GATE_SIGMOID) {
    const float x = fminf(fmaxf(-g, -126.f), 126.f);       // (a NaN gate is let through below)
    const float t = __fmul_rn(x, 1.44269504f), d = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -t));
    return g != g ? g : __fdividef(1.f, fmaf(fast_exp2(t), fmaf(d, 0.693147181f, 1.f), 1.f));
  }
  return act == TQ_GATE_TANH ? tanhf(g) : g;
}

// Sum over the T threads of a row: a warp by itself, or a CTA through `part`, whose
// two halves take turns, so that one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float x, int T, float (*part)[32], int& turn) {
  x = warp_sum(x);
  if (T == 32) return x;
  const int lane = threadIdx.x & 31;
  if (lane == 0) part[turn][threadIdx.x >> 5] = x;
  __syncthreads();
  // a partial sum a lane: read one after the other by every thread, 16 of them were half of a
  // row's instructions
  x = warp_sum(lane < T / 32 ? part[turn][lane] : 0.f);
  turn ^= 1;
  return x;
}

// Offset of a row.
__device__ __forceinline__ int64_t row_at(const NormParams& p, const int64_t (&s)[4], uint32_t r) {
  if (p.n2 == 0) return r * s[2];
  const uint32_t n1 = (uint32_t)p.n1, n2 = (uint32_t)p.n2, i01 = r / n2, i0 = i01 / n1;
  return i0 * s[0] + (i01 - i0 * n1) * s[1] + (r - i01 * n2) * s[2];
}

using tc::f2;

// The common case: rows of up to 8,192 values in chunks of V = 8 or 2 neighbours.  T threads
// (a warp, or the CTA) take row after row, 8 values each, with what a column needs in
// registers in 32 bits, gate and scale folded in:
//   y = residual + (x r) A + B,   h = (y r') C + D
// (A = (w + offset) F, B = b F, F = scale act(gate); with a gate per element the products
// with F are made where it is used, to the same bits: a row alone, whose gate is either, is the
// row of a batch), and the next rows' values on their way: two with chunks of 8 (16,381 rows of 4,096: one
// 144 us, two 117), one with chunks of 2, whose registers leave less room (2,051 rows of
// 2,050: 33 us, 41).  GE: a gate per element, BIAS: B and D.  The
// arithmetic, on fp32 pairs, is 6 instructions a value without a gate per element.
// residual_norm_kernel below goes through the same roundings.
template <int XT, int RT, int V, bool GE, bool BIAS, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_norm_rows_kernel(NormParams p, int T) {
  constexpr int NK = 8 / V, NP = 4;                        // chunks and pairs of a thread
  constexpr bool TWO = V == 8;                             // rows on their way
  __shared__ float part[2][32];
  int turn = 0;
  const int t = threadIdx.x % T;
  const uint32_t per = blockDim.x / T, step = gridDim.x * per, rows = (uint32_t)p.rows;
  uint32_t row = blockIdx.x * per + threadIdx.x / T;
  if (row >= rows) return;                                 // whole warps where a row is one's
  auto col = [&](int k) { return (k * T + t) * V; };
  auto inside = [&](int k) { return col(k) < p.C; };       // C is a multiple of V
  struct Raw {
    Chunk<XT, V> x[NK];
    Chunk<RT, V> r[NK];
    uint32_t g[GE ? NK : 1][V / 2];                        // a gate of 16 bits
  };
  auto fetch = [&](Raw& w, uint32_t r) {
    const int64_t xb = row_at(p, p.xs, r), rb = row_at(p, p.rs, r), gb = GE ? row_at(p, p.gs, r) : 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      w.x[k].clear();
      w.r[k].clear();
      if (!inside(k)) continue;
      w.x[k].load(p.x, xb + col(k));
      w.r[k].load(p.r, rb + col(k));
      if constexpr (GE) {
        Chunk<TQ_F16, V> g;
        g.load(p.g, gb + col(k));
#pragma unroll
        for (int i = 0; i < V / 2; ++i) w.g[k][i] = g.w[i];
      }
    }
  };
  Raw cur, nxt;
  fetch(cur, row);
  if (TWO && rows - row > step) fetch(nxt, row + step);
  // a column's factors
  f2 A[NP], B[BIAS ? NP : 1], C[NP], D[BIAS ? NP : 1];
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    float a[V], b[V], c[V], d[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { a[e] = c[e] = 1.f; b[e] = d[e] = 0.f; }
    if (inside(k)) {
      auto param = [&](float (&v)[V], const void* base, int dtype, float add) {
        if (!base) return;
        load_param<V>(v, base, dtype, col(k));
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += add;
      };
      param(a, p.post.w, p.post.dtype, p.post.offset);
      param(c, p.pre.w, p.pre.dtype, p.pre.offset);
      if (BIAS) {
        param(b, p.post.b, p.post.dtype, 0.f);
        param(d, p.pre.b, p.pre.dtype, 0.f);
      }
      float g[V];
      const bool channel = !GE && p.gmode == 1;            // one for all rows
      if (channel) load_param<V>(g, p.g, p.gd, col(k));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f = GE ? 1.f : p.scale * (channel ? activate(g[e], p.act) : 1.f);
        a[e] *= f;
        b[e] *= f;
      }
    }
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const int i = (k * V + e) / 2;
      A[i] = tc::f2_make(a[e], a[e + 1]);
      C[i] = tc::f2_make(c[e], c[e + 1]);
      if constexpr (BIAS) {
        B[i] = tc::f2_make(b[e], b[e + 1]);
        D[i] = tc::f2_make(d[e], d[e + 1]);
      }
    }
  }
  const float inv_c = 1.f / (float)p.C;
  const f2 zero = tc::f2_make(0.f, 0.f);
  auto pair_sum = [](f2 x) {
    float lo, hi;
    tc::f2_split(x, lo, hi);
    return lo + hi;
  };
  for (;;) {
    Raw far;
    if (TWO) {
      if (rows - row > 2 * (uint64_t)step) fetch(far, row + 2 * step);
    } else if (rows - row > step) {
      fetch(nxt, row + step);
    }
    f2 v[NP];
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
      for (int e = 0; e < V; e += 2) v[(k * V + e) / 2] = cur.x[k].pair(e);
    // takes the mean off (where the norm does) and returns the factor
    auto norm = [&](const NormSide& n) {
      if (n.centered) {
        f2 sum = v[0];
        const f2 one = tc::f2_make(1.f, 1.f);
#pragma unroll
        for (int i = 1; i < NP; ++i) sum = tc::f2_fma(v[i], one, sum);
        const float mean = row_sum(pair_sum(sum), T, part, turn) * inv_c;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          const f2 m = inside(k) ? tc::f2_make(-mean, -mean) : zero;
#pragma unroll
          for (int i = k * V / 2; i < (k + 1) * V / 2; ++i) v[i] = tc::f2_fma(m, one, v[i]);
        }
      }
      f2 ss = tc::f2_mul(v[0], v[0]);
#pragma unroll
      for (int i = 1; i < NP; ++i) ss = tc::f2_fma(v[i], v[i], ss);
      return 1.f / sqrtf(fmaf(row_sum(pair_sum(ss), T, part, turn), inv_c, n.eps));
    };
    const float r1 = p.post.on ? norm(p.post) : 1.f;
    const f2 rr = tc::f2_make(r1, r1);
    float one = 1.f;
    if (!GE && p.gmode == 2) one = activate(load_elem(p.g, p.gd, row_at(p, p.gs, row)), p.act);
    const int64_t yb = row_at(p, p.ys, row);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const int i = (k * V + e) / 2;
        const f2 res = cur.r[k].pair(e);
        f2 z = tc::f2_mul(v[i], rr);
        if constexpr (GE) {
          const uint32_t u = cur.g[k][e / 2];
          float lo, hi;
          if (p.gd == TQ_F16) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&u));
            lo = h.x; hi = h.y;
          } else {
            lo = __uint_as_float(u << 16);
            hi = __uint_as_float(u & 0xFFFF0000u);
          }
          const f2 f = tc::f2_mul(tc::f2_make(p.scale, p.scale),
                                  tc::f2_make(activate(lo, p.act), activate(hi, p.act)));
          if constexpr (BIAS) {
            z = tc::f2_fma(z, tc::f2_mul(A[i], f), tc::f2_mul(B[i], f));
            v[i] = tc::f2_fma(z, tc::f2_make(1.f, 1.f), res);
          } else {
            v[i] = tc::f2_fma(z, tc::f2_mul(A[i], f), res);
          }
        } else if (p.gmode == 2) {
          z = BIAS ? tc::f2_fma(z, A[i], B[i]) : tc::f2_mul(z, A[i]);
          v[i] = tc::f2_fma(z, tc::f2_make(one, one), res);
        } else if constexpr (BIAS) {
          const f2 zb = tc::f2_fma(z, A[i], B[i]);
          v[i] = tc::f2_fma(zb, tc::f2_make(1.f, 1.f), res);
        } else {
          v[i] = tc::f2_fma(z, A[i], res);
        }
        if (!inside(k)) v[i] = zero;
        tc::f2_split(v[i], o[e], o[e + 1]);
      }
      if (inside(k)) Chunk<RT, V>::store(p.y, yb + col(k), o);
    }
    if (p.h) {
      const float r2 = norm(p.pre);
      const f2 r2r = tc::f2_make(r2, r2);
      const int64_t hb = row_at(p, p.hs, row);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const int i = (k * V + e) / 2;
          f2 z = tc::f2_mul(v[i], r2r);
          z = BIAS ? tc::f2_fma(z, C[i], D[i]) : tc::f2_mul(z, C[i]);
          tc::f2_split(z, o[e], o[e + 1]);
        }
        if (inside(k)) Chunk<XT, V>::store(p.h, hb + col(k), o);
      }
    }
    if (rows - row <= step) return;
    row += step;
    cur = nxt;
    if (TWO) nxt = far;
  }
}

using NormFn = void (*)(NormParams, int);

// Up to 384 threads no instance spills, at 64 to 118 registers.  Above,
// two CTAs of 512 threads an SM leave 64: rows of 16 bits without biases and gates per element fit,
// layer norms spill 80 bytes a thread, with a gate of their own 164, with an fp32 residual 28
// to 272, fp32 throughout 68 to 348.  8,192 rows of 4,096: bf16 layer norms 98 us for 268 MB
// (2.7 TB/s), an fp32 residual 84 for 403 MB (4.8), a gate per element 87 for 336 MB (3.8), that
// with layer norms 139.
template <int XT, int RT, int V>
NormFn rows_fn(bool ge, bool bias, bool wide) {
#define TQ_ROWS(GE, BIAS) \
  if (ge == GE && bias == BIAS) \
    return wide ? residual_norm_rows_kernel<XT, RT, V, GE, BIAS, 1024> : residual_norm_rows_kernel<XT, RT, V, GE, BIAS, 384>;
  TQ_ROWS(false, false) TQ_ROWS(false, true) TQ_ROWS(true, false) TQ_ROWS(true, true)
#undef TQ_ROWS
  return nullptr;
}

template <int XT>
NormFn rows_fn_x(int rd, int v, bool ge, bool bias, bool wide) {
#define TQ_ROWS(RT) \
  if (rd == RT) return v == 8 ? rows_fn<XT, RT, 8>(ge, bias, wide) : rows_fn<XT, RT, 2>(ge, bias, wide);
  TQ_ROWS(TQ_F32) TQ_ROWS(TQ_F16) TQ_ROWS(TQ_BF16)
#undef TQ_ROWS
  return nullptr;
}

// Everything else: rows above 8,192 values (more than 1,024 threads' 8), views whose rows start on
// odd elements, and fp32 gates per element, eight registers a row on its way more than the
// instances above have.  T threads per row (a warp, or the CTA), 8 VPT values each in chunks of V
// neighbours; V = 1 takes any stride.  8,192 fp32 rows of 4,096 with fp32 gates 152 us for 671
// MB (4.4 TB/s), 2,048 bf16 rows of 16,384 with gates 142 (2.4), 2,048 of 4,097 111.  Sums and products go in the order of the kernel above,
// even and odd values by themselves, and no product joins a sum but by fmaf: a gate of 32 bits
// per element (whose rows on their way the registers above have no room for) gives the bits
// that a gate of the channels gives there.
template <int XT, int RT, int VPT, int V>
__global__ void __launch_bounds__(VPT == 1 ? 1024 : 512) residual_norm_kernel(NormParams p, int T) {
  constexpr int NK = 8 * VPT / V;                          // chunks of a thread
  __shared__ float part[2][32];
  int turn = 0;
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / T) + threadIdx.x / T;
  if (row >= p.rows) return;                               // whole warps where a row is one's
  auto at = [&](const int64_t (&s)[4]) { return row_at(p, s, (uint32_t)row); };
  const int64_t xb = at(p.xs), rb = at(p.rs);
  // values of chunk k: from column c(k) on
  auto col = [&](int k) { return (k * T + t) * V; };
  auto inside = [&](int k) { return col(k) < p.C; };       // C is a multiple of V
  auto place = [&](const int64_t (&s)[4], int k) { return V == 1 ? col(k) * s[3] : (int64_t)col(k); };
  Chunk<XT, V> xr[NK];
  Chunk<RT, V> rr[NK];
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    xr[k].clear();
    rr[k].clear();
    if (inside(k)) {
      xr[k].load(p.x, xb + place(p.xs, k));
      rr[k].load(p.r, rb + place(p.rs, k));
    }
  }
  // a gate per element, on its way beside them where there are registers
  constexpr bool EARLY = VPT == 1;
  const int64_t gb = p.gmode ? at(p.gs) : 0;
  float early[EARLY ? NK : 1][V];
  if (EARLY && p.gmode == 1)
#pragma unroll
    for (int k = 0; k < NK; ++k)
      if (inside(k)) load_param<V>(early[k], p.g, p.gd, gb + place(p.gs, k));
  float v[NK][V];
#pragma unroll
  for (int k = 0; k < NK; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) v[k][e] = xr[k].get(e);
  const float inv_c = 1.f / (float)p.C;
  auto val = [&](int i) -> float& { return v[i / V][i % V]; };
  // takes the mean off (where the norm does) and returns the factor
  auto norm = [&](const NormSide& s) {
    if (s.centered) {
      float lo = val(0), hi = val(1);
#pragma unroll
      for (int i = 2; i < 8 * VPT; i += 2) {
        lo = __fadd_rn(lo, val(i));
        hi = __fadd_rn(hi, val(i + 1));
      }
      const float mean = __fmul_rn(row_sum(__fadd_rn(lo, hi), T, part, turn), inv_c);
#pragma unroll
      for (int k = 0; k < NK; ++k)
        if (inside(k))
#pragma unroll
          for (int e = 0; e < V; ++e) v[k][e] = __fsub_rn(v[k][e], mean);
    }
    float lo = __fmul_rn(val(0), val(0)), hi = __fmul_rn(val(1), val(1));
#pragma unroll
    for (int i = 2; i < 8 * VPT; i += 2) {
      lo = fmaf(val(i), val(i), lo);
      hi = fmaf(val(i + 1), val(i + 1), hi);
    }
    return 1.f / sqrtf(fmaf(row_sum(__fadd_rn(lo, hi), T, part, turn), inv_c, s.eps));
  };
  // weights and biases of chunk k
  auto params = [&](const NormSide& s, int k, float (&w)[V], float (&b)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) { w[e] = 1.f; b[e] = 0.f; }
    if (s.w) {
      load_param<V>(w, s.w, s.dtype, col(k));
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] += s.offset;
    }
    if (s.b) load_param<V>(b, s.b, s.dtype, col(k));
  };
  const bool bias = p.post.b || p.pre.b;
  const float r1 = p.post.on ? norm(p.post) : 1.f;
  const float one = p.gmode == 2 ? p.scale * activate(load_elem(p.g, p.gd, gb), p.act) : p.scale;
  const int64_t yb = at(p.ys);
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    if (!inside(k)) continue;
    float g[V], w[V], b[V];
    params(p.post, k, w, b);
    if (!EARLY && p.gmode == 1) load_param<V>(g, p.g, p.gd, gb + place(p.gs, k));
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x = EARLY ? early[EARLY ? k : 0][e] : g[e];
      const float f = p.gmode == 1 ? __fmul_rn(p.scale, activate(x, p.act)) : one;
      const float z = __fmul_rn(v[k][e], r1), a = __fmul_rn(w[e], f), res = rr[k].get(e);
      v[k][e] = bias ? __fadd_rn(fmaf(z, a, __fmul_rn(b[e], f)), res) : fmaf(z, a, res);
    }
    Chunk<RT, V>::store(p.y, yb + place(p.ys, k), v[k]);
  }
  if (!p.h) return;
  const float r2 = norm(p.pre);
  const int64_t hb = at(p.hs);
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    if (!inside(k)) continue;
    float w[V], b[V];
    params(p.pre, k, w, b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float z = __fmul_rn(v[k][e], r2);
      v[k][e] = bias ? fmaf(z, w[e], b[e]) : __fmul_rn(z, w[e]);
    }
    Chunk<XT, V>::store(p.h, hb + place(p.hs, k), v[k]);
  }
}

template <int XT, int RT>
NormFn norm_fn(int vpt, int v) {
#define TQ_NORM(N, V) if (vpt == N && v == V) return residual_norm_kernel<XT, RT, N, V>;
  TQ_NORM(1, 8) TQ_NORM(4, 8) TQ_NORM(8, 8)
  TQ_NORM(1, 2) TQ_NORM(4, 2) TQ_NORM(8, 2)
  TQ_NORM(1, 1) TQ_NORM(2, 1) TQ_NORM(4, 1) TQ_NORM(8, 1)
#undef TQ_NORM
  return nullptr;
}

template <int XT>
NormFn norm_fn_x(int rd, int vpt, int v) {
  return rd == TQ_F32 ? norm_fn<XT, TQ_F32>(vpt, v)
         : rd == TQ_F16 ? norm_fn<XT, TQ_F16>(vpt, v) : norm_fn<XT, TQ_BF16>(vpt, v);
}

NormSide norm_side(const tq_row_norm* n) {
  NormSide s = {};
  if (!n) return s;
  s.on = 1;
  s.centered = n->centered;
  s.dtype = n->dtype;
  s.w = n->weight;
  s.b = n->bias;
  s.eps = n->eps;
  s.offset = n->offset;
  return s;
}

// Are rows of the view read and written v neighbours at a time?  By the strides as they are
// given, those of single entries too: a row taken out of a batch by slicing goes like the batch.
bool takes_chunks(const tq_tensor4* x, int v) {
  const int bytes = tmin(16, v * (x->dtype == TQ_F32 ? 4 : 2));
  const int es = x->dtype == TQ_F32 ? 4 : 2;
  if (x->shape[3] % v || (x->shape[3] > 1 && x->stride[3] != 1) ||
      reinterpret_cast<uintptr_t>(x->data) % bytes)
    return false;
  for (int i = 0; i < 3; ++i)
    if ((x->stride[i] * es) % bytes) return false;
  return true;
}

bool param_takes_chunks(const tq_row_norm* n, int v) {
  if (!n) return true;
  const int bytes = tmin(16, v * (n->dtype == TQ_F32 ? 4 : 2));
  return (reinterpret_cast<uintptr_t>(n->weight) | reinterpret_cast<uintptr_t>(n->bias)) % bytes == 0;
}

}  // namespace

int launch_residual_norm(const tq_residual_norm_args* a, cudaStream_t st) {
  NormParams p = {};
  const tq_tensor4 *x = a->x, *r = a->residual, *g = a->gate;
  p.rows = x->shape[0] * x->shape[1] * x->shape[2];
  if (p.rows == 0) return TQ_OK;
  p.n1 = x->shape[1];
  p.n2 = x->shape[2];
  p.C = (int)x->shape[3];
  p.x = x->data;
  p.r = r->data;
  p.y = a->residual_out->data;
  p.h = a->pre ? a->out->data : nullptr;
  for (int i = 0; i < 4; ++i) {
    p.xs[i] = x->stride[i];
    p.rs[i] = r->stride[i];
    p.ys[i] = a->residual_out->stride[i];
    if (p.h) p.hs[i] = a->out->stride[i];
    if (g) p.gs[i] = g->stride[i];
  }
  if (g) {
    p.g = g->data;
    p.gd = g->dtype;
    p.gmode = g->stride[3] == 0 ? 2 : 1;
    p.act = a->gate_act;
  }
  // leading dims that are one run of rows in every tensor
  bool flat = true;
  for (const tq_tensor4* z : {x, r, g, a->residual_out, p.h ? a->out : nullptr})
    for (int i = 0; z && i < 2; ++i)
      flat = flat && (z->shape[i] == 1 || z->stride[i] == z->stride[2] * (i ? z->shape[2] : z->shape[1] * z->shape[2]));
  if (flat) p.n2 = 0;
  p.scale = a->scale;
  p.post = norm_side(a->post);
  p.pre = norm_side(a->pre);
  int v = 1;
  for (int c : {8, 2}) {
    if (takes_chunks(x, c) && takes_chunks(r, c) && takes_chunks(a->residual_out, c) &&
        (!p.h || takes_chunks(a->out, c)) && (p.gmode != 1 || takes_chunks(g, c)) &&
        param_takes_chunks(a->post, c) && param_takes_chunks(a->pre, c)) {
      v = c;
      break;
    }
  }
  const int units = (p.C + 7) / 8;
  // a gate that differs from row to row (what a single row's gate is, its bits do not say)
  bool per_row = false;
  for (int i = 0; g && i < 3; ++i) per_row = per_row || (g->shape[i] > 1 && g->stride[i] != 0);
  const bool ge = p.gmode == 1 && per_row;
  if (v > 1 && units <= 1024 && !(ge && p.gd == TQ_F32)) {
    const bool bias = p.post.b || p.pre.b;
    const int T = (units + 31) & ~31, per = T == 32 ? 4 : 1;
    const bool wide = T > 384;
    const NormFn fn = x->dtype == TQ_F32   ? rows_fn_x<TQ_F32>(r->dtype, v, ge, bias, wide)
                      : x->dtype == TQ_F16 ? rows_fn_x<TQ_F16>(r->dtype, v, ge, bias, wide)
                                           : rows_fn_x<TQ_BF16>(r->dtype, v, ge, bias, wide);
    int64_t grid = (p.rows + per - 1) / per;
    if (grid > device_sm_count())
      grid = tmin(grid, (int64_t)device_sm_count() * occupancy((const void*)fn, T * per, 0));
    fn<<<(unsigned)grid, T * per, 0, st>>>(p, T);
    return check_launch("tq_residual_norm");
  }
  // Threads of a row and their values, 8 vpt each, by the width (and chunks, those of the kernel
  // above) alone: a row's sums do not depend on how many rows come with it.
  int vpt, T;
  if (v > 1 && units <= 1024) {
    vpt = 1;
    T = (units + 31) & ~31;
  } else if (units <= 128) {
    T = 32;
    vpt = units <= 32 ? 1 : units <= 64 ? 2 : 4;
  } else {
    vpt = units <= 1024 ? 1 : units <= 2048 ? 4 : 8;
    T = ((units + vpt - 1) / vpt + 31) & ~31;
  }
  const NormFn fn = x->dtype == TQ_F32   ? norm_fn_x<TQ_F32>(r->dtype, vpt, v)
                    : x->dtype == TQ_F16 ? norm_fn_x<TQ_F16>(r->dtype, vpt, v)
                                         : norm_fn_x<TQ_BF16>(r->dtype, vpt, v);
  const int per = T == 32 ? 4 : 1;
  const int64_t grid = (p.rows + per - 1) / per;
  fn<<<(unsigned)grid, T * per, 0, st>>>(p, T);
  return check_launch("tq_residual_norm");
}

}  // namespace tq
