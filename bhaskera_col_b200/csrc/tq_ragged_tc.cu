// tq_ragged_tc.cu — ragged append and ragged read-back on the 5th-generation
// tensor cores (head_dim 64 and 128); other shapes run the CUDA-core kernels of
// tq_ragged.cu, which give the math.
//
// A tile is 128 consecutive head vectors of the flattened batch (token-major,
// so the heads of a token share its row of the rotation table and a tile is
// contiguous in memory), M of one tcgen05.mma with N = K = head_dim.  One
// persistent CTA per SM, a launch each for K and V, four roles:
//   makers      operand of the next tile.  Append (16 warps): load, norm,
//               rotate, norm again, split into fp16; read-back (8 warps): codes
//               -> centroids through lane-replicated tables.  They fetch one
//               tile ahead of what they make.
//   locators    two warps find each vector's request, position and page
//   issuer      one thread issues the MMAs into one of two accumulators
//   epilogue    one thread per vector and 32 columns at a time.  Append (8
//               warps): bucketize and pack; read-back (4 per 32 columns): times
//               the norm, out through shared memory so that rows leave in
//               whole lines
//
// Append: y n s 2^6 = (x s) (2^6 R)^T with s the power of two that puts ||x||
// into [2^10, 2^11), x s = hi + lo and 2^6 R = hi + lo in fp16 (22 bits, the
// scales keep lo out of the subnormals), fp32 accumulation:
//   hi hi + hi lo, and + lo hi where x has more than fp16's bits (fp32 inputs,
//   a normed or rotated k; a bf16 or fp16 x is its own hi).
// R's rows lie in the packed order of the row (K quad order, V octet order), so
// accumulator column p is the coordinate stored at position p.
// Bucketize without branches, exactly: a cell of the grid 0.4 x the smallest
// gap wide holds at most one boundary in its window, so the cell's entry {-b
// 2^100, codes below} and the sign of y - b give the code (the same scheme as
// tq_append_tc.cu).  Tables that do not fit take a binary search.
//
// Read-back: x = (c R) n with R's rows in packed order as the K dimension,
// c and R as fp16 hi + lo (three products); for bf16 results c = hi alone: its
// rounding, 2^-12 of each term on average, is an eighth of the result's own and
// takes their error from 1.66e-3 to 1.68e-3, one bf16 step in 5 % of the values.  lo
// too would leave room for one operand tile in flight instead of two (17,971 tokens
// 58.5 us against 50); who wants it asks for fp32 results.
//
// Bounds: HBM (256 B in, 66 out per 4-bit vector of 128 bf16, or the reverse);
// in fact a role's instructions per tile: append's makers (3 us a tile: norms,
// rotation, split) and epilogue (2 us: 9 instructions a coordinate), read-back's
// epilogue (3.2 us).  Measured, K and V: append of 11,272 tokens x 8 heads of 128,
// 4-bit, with norm and rotation, and reading them back 103 us for 122 MB (half of
// it each); read-back of 17,971 tokens 50 us for 93 MB, 1.9 TB/s; a launch of
// few tiles 8-10 us, set-up (rotation, tables) and one tile's latency.
//
// Every wait is bounded; on expiry the kernel sets TQ_DEV_WAIT_TIMEOUT in the
// status word, no MMA is left in flight and tensor memory is released.
#include "tq_internal.h"
#include "tq_ragged.cuh"
#include "tq_tc.cuh"

#include <limits.h>
#include <type_traits>

namespace tq {
namespace {

constexpr int kM = 128;                    // vectors per tile
constexpr int kRing = 4;                   // tiles of per-vector data in flight
constexpr int kSmem = 227 * 1024;
constexpr float kCmp = 1.2676506e30f;      // 2^100
constexpr float kRScale = 64.f;
// Append: a coordinate of the unit vector R x / ||x|| this near to a boundary is
// computed again in 64 bits, so that the codes are those of exact arithmetic.
// The operands' 22 bits and the sums' rounding leave the first value a few 1e-8
// off (one code in 600,000 came out wrong); 3e-7 is several times that and takes
// one coordinate in 50,000 (128 dims, 4 bits).
constexpr float kNear = 3e-7f;

// i / d for 0 <= i < 2^31 as a product: m = ceil(2^(31 + s) / d), 2^s >= d.
struct FastDiv {
  uint32_t m, s;
  int d;
  __device__ __forceinline__ int div(int i) const {
    return (int)(((uint64_t)(uint32_t)i * m) >> (31 + s));
  }
};
FastDiv fast_div(int d) {
  FastDiv f;
  f.d = d;
  f.s = 0;
  while ((1 << f.s) < d) ++f.s;
  f.m = (uint32_t)((((uint64_t)1 << (31 + f.s)) + d - 1) / d);
  return f;
}

struct RaggedTc {
  PageGeom g;
  const float* cent[2];
  const float* bnd[2];
  const float* rot;                        // R [D][D]
  uint8_t* pages;
  PageMap pm;
  uint32_t* status;
  RaggedView rv;
  int H, ntiles, nvec;                     // heads, tiles, vectors (rows x heads)
  FastDiv by_h;
  const void* x[2];                        // append: inputs; read-back: outputs (NULL: absent)
  int dtype[2];
  int64_t stride[2][3];                    // head, row, dim
  int vec[2];                              // read-back: rows take 16-byte stores
  int use_lo[2];                           // append: x has more bits than fp16
  HeadXform f;                             // of K (append)
  const void* pos; int pos64; int64_t pos_stride;
};

// MAKERS maker warps (kM / MAKERS vectors each), the issuing warp, two
// locators, SPLIT epilogue warps per lane quarter of tensor memory.
template <int D, int MAKERS, int SPLIT>
struct Roles {
  static constexpr int kMakers = MAKERS, kVecs = kM / MAKERS, kSplit = SPLIT, kEpi = 4 * SPLIT;
  static constexpr int kIssuer = MAKERS, kLocators = MAKERS + 1, kEpi0 = MAKERS + 3;
  static constexpr int kThreads = 32 * (kEpi0 + kEpi);
};
// Making an append operand (norms, rotation, split) takes twice its epilogue's
// instructions, a read-back operand half of it.
template <int D> using AppendRoles = Roles<D, 16, 2>;
template <int D> using ReadRoles = Roles<D, 8, D / 32>;

template <int D>
struct Shape {
  static constexpr int kTerm = kM * D * 2;                 // one fp16 operand tile
  static constexpr int kB = D * D * 2;                     // one term of R
};

// Byte offset of 16-byte chunk c of row r: [64-column half][rows][128 B], swizzled.
template <int ROWS>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void expired(uint32_t* status, volatile int* abort_flag) {
  *abort_flag = 1;
  atomicOr(status, TQ_DEV_WAIT_TIMEOUT);
}

// Bounded wait (2 s) that also ends once another role has given up.  No
// suspend-time hint: a hinted wait of the issuing thread resumed up to 2 us
// late, twice a tile's MMAs.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                         uint32_t* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*abort_flag) return false;
      const uint64_t t = global_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 > 2000000000ull) break;
    }
  }
  expired(status, abort_flag);
  return false;
}

__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_half2(a, b);
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  lo = pack_half2(a - __low2float(h), b - __high2float(h));
}

// R's rows in packed order, times kRScale, as fp16 hi at `b` and lo behind it,
// by N threads with all their loads in flight.
template <int D, int N>
__device__ __forceinline__ void stage_rotation(unsigned char* b, const float* rot, int which,
                                               int tid) {
  constexpr int IT = (D * D / 8 + N - 1) / N;
  float4 u[IT], v[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int i = tid + k * N;
    if (i >= D * D / 8) break;
    const int r = i / (D / 8), c = i % (D / 8);
    const int row = which == 0 ? k_coord_at(r, D) : v_coord_at(r, D);
    const float4* src = reinterpret_cast<const float4*>(rot + row * D + 8 * c);
    u[k] = __ldg(src);
    v[k] = __ldg(src + 1);
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int i = tid + k * N;
    if (i >= D * D / 8) break;
    uint32_t h[4], l[4];
    split_pair(u[k].x * kRScale, u[k].y * kRScale, h[0], l[0]);
    split_pair(u[k].z * kRScale, u[k].w * kRScale, h[1], l[1]);
    split_pair(v[k].x * kRScale, v[k].y * kRScale, h[2], l[2]);
    split_pair(v[k].z * kRScale, v[k].w * kRScale, h[3], l[3]);
    const uint32_t at = chunk_at<D>(i / (D / 8), i % (D / 8));
    *reinterpret_cast<uint4*>(b + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(b + Shape<D>::kB + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// A tile's vectors, one ring entry: where they lie (locators) and what the
// makers leave for the epilogue.
struct Vecs {
  uint8_t* page[kM];                       // NULL: no place
  int slot[kM];                            // token in its page
  int row[kM];                             // row of the rotation table; several axes: of the batch, -1: no place
  float n[kM];                             // norm
  float inv[kM];                           // append: factor of the accumulator
  uint8_t state[kM];                       // 0: row of no request, 1: no place, 2: stored
};

// The batch's offsets and lengths in shared memory where they fit (a search
// over global memory costs a trip to L2 per step: 6 us for 64 requests).
constexpr int kStaged = 512;
struct Requests {
  const int32_t* q_start;
  const int32_t* seq_lens;
};
constexpr int kStagedBytes = (2 * kStaged + 4) * 4;

__device__ __forceinline__ Requests stage_requests(const RaggedView& v, unsigned char* at, int tid,
                                                   int nthreads) {
  Requests q = {v.q_start, v.seq_lens};
  if (v.R <= kStaged) {
    int32_t* s = reinterpret_cast<int32_t*>(at);
    for (int i = tid; i <= v.R; i += nthreads) s[i] = __ldg(v.q_start + i);
    for (int i = tid; i < v.R; i += nthreads) s[kStaged + 4 + i] = __ldg(v.seq_lens + i);
    q.q_start = s;
    q.seq_lens = s + kStaged + 4;
  }
  return q;
}

// Shared pieces of both kernels: barriers, the issuing thread, the accumulators.
struct Pipe {
  uint64_t* a_full;                        // [2] maker warps
  uint64_t* a_empty;                       // [2] MMA commit
  uint64_t* acc_full;                      // [2] MMA commit
  uint64_t* acc_empty;                     // [2] epilogue warps
  uint64_t* loc_full;                      // [kRing] locators: the tile's places are known
  uint64_t* loc_free;                      // [kRing] epilogue warps
  volatile int* abort_flag;
  uint32_t* tmem_slot;
};

__device__ __forceinline__ Pipe make_pipe(unsigned char* at) {
  uint64_t* b = reinterpret_cast<uint64_t*>(at);
  Pipe p;
  p.a_full = b;
  p.a_empty = b + 2;
  p.acc_full = b + 4;
  p.acc_empty = b + 6;
  p.loc_full = b + 8;
  p.loc_free = b + 8 + kRing;
  p.tmem_slot = reinterpret_cast<uint32_t*>(b + 8 + 2 * kRing);
  p.abort_flag = reinterpret_cast<volatile int*>(b + 9 + 2 * kRing);
  return p;
}
constexpr int kPipeBytes = 192;            // with 16 bytes of the lookup grid at its end

__device__ __forceinline__ void init_pipe(const Pipe& p, int makers, int epi_warps) {
  for (int i = 0; i < 2; ++i) {
    mbar_init(&p.a_full[i], makers);
    mbar_init(&p.a_empty[i], 1);
    mbar_init(&p.acc_full[i], 1);
    mbar_init(&p.acc_empty[i], epi_warps);
  }
  for (int i = 0; i < kRing; ++i) {
    mbar_init(&p.loc_full[i], 2);
    mbar_init(&p.loc_free[i], epi_warps);
  }
  *p.abort_flag = 0;
  fence_mbar_init();
}

// Two warps, half a tile each: two vectors per lane.  A vector's place is a
// chain of dependent loads (offsets, length, block table); found by warps of
// their own and up to kRing tiles ahead, the chain delays nobody.  AXES: a stored
// vector's row is that of its positions, which nobody looks up for any other.
template <bool AXES>
__device__ __forceinline__ void locate_tiles(const RaggedTc& p, const Pipe& pp, Vecs* ring,
                                             const Requests& rq, int half, int first, int step) {
  constexpr int NV = kM / 64;
  const int lane = threadIdx.x & 31, R = (int)p.rv.R;
  int it = 0;
  for (int tile = first; tile < p.ntiles; tile += step, ++it) {
    const int e = it % kRing;
    const bool ok = it < kRing || wait_for(&pp.loc_free[e], (uint32_t)(((it / kRing) - 1) & 1),
                                           pp.abort_flag, p.status);
    if (!__all_sync(0xffffffffu, ok)) break;
    int64_t pos[NV], entry[NV], to[NV];
    int n[NV], state[NV];
    const int begin = rq.q_start[0], end = rq.q_start[R];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = tile * kM + 64 * half + 32 * k + lane;
      n[k] = p.by_h.div(i);
      const int h = i - n[k] * p.H;
      state[k] = i < p.nvec && n[k] >= begin && n[k] < end;
      int lo = 0, hi = R;                  // q_start[lo] <= n < q_start[hi] at the end
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (rq.q_start[mid] <= n[k]) lo = mid; else hi = mid;
      }
      pos[k] = (int64_t)rq.seq_lens[lo] - rq.q_start[lo + 1] + n[k];
      const bool in = state[k] && pos[k] >= 0 && pos[k] < p.rv.cap;
      if (state[k] && !in) atomicOr(p.status, TQ_DEV_BAD_POSITION);
      entry[k] = in ? page_entry(p.pm, (int64_t)lo * p.H + h, pos[k] / kPageTokens) : -1;
      to[k] = pos[k];
      if (!AXES && p.pos && in)
        to[k] = p.pos64
                    ? (int64_t)__ldg(reinterpret_cast<const long long*>(p.pos) + n[k] * p.pos_stride)
                    : (int64_t)__ldg(reinterpret_cast<const int*>(p.pos) + n[k] * p.pos_stride);
      if (in) state[k] = 2;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = 64 * half + 32 * k + lane;
      if (state[k] == 2 && !entry_ok(p.pm, entry[k])) {
        atomicOr(p.status, TQ_DEV_BAD_BLOCK);
        state[k] = 1;
      }
      const bool in = state[k] == 2;
      ring[e].page[at] = in ? p.pages + entry[k] * (int64_t)p.g.page_bytes : nullptr;
      ring[e].slot[at] = (int)(pos[k] & (kPageTokens - 1));
      ring[e].row[at] = AXES ? (in ? n[k] : -1) : in && p.f.cos_sin ? (int)table_row(p.f, to[k], p.status) : 0;
      ring[e].state[at] = (uint8_t)state[k];
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive_cta(&pp.loc_full[e]);
  }
}

// One thread: the MMAs of every tile.  terms(stage, term, a, b) gives the
// operand addresses of each product or false past the last.
template <int D, int STAGES, bool B_MN, class Terms>
__device__ __forceinline__ void issue_tiles(const Pipe& pp, uint32_t tmem, int first, int step,
                                            int ntiles, uint32_t* status, Terms terms) {
  constexpr uint32_t idesc = tc::idesc_f16_f32(kM, D) | (B_MN ? 1u << 16 : 0u);
  int it = 0, issued = 0;
  for (int tile = first; tile < ntiles; tile += step, ++it) {
    const int st = it % STAGES, ac = it & 1;
    if (!wait_for(&pp.a_full[st], (uint32_t)((it / STAGES) & 1), pp.abort_flag, status) ||
        (it >= 2 &&
         !wait_for(&pp.acc_empty[ac], (uint32_t)(((it / 2) - 1) & 1), pp.abort_flag, status)))
      break;
    tc::tc_fence_after();
    uint32_t a, b;
    for (int term = 0; terms(st, term, a, b); ++term)
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t ad =
            tc::sdesc_kmajor_sw128(a + (uint32_t)((ks >> 2) * (kM * 128) + (ks & 3) * 32));
        uint64_t bd;
        if (B_MN) {
          // 16 rows of K on; N blocks of 64 columns D x 128 B apart
          bd = tc::sdesc_kmajor_sw128(b + ks * 2048);
          bd = (bd & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)((D * 128) >> 4) << 16);
        } else {
          bd = tc::sdesc_kmajor_sw128(b + (uint32_t)((ks >> 2) * (D * 128) + (ks & 3) * 32));
        }
        tc::umma_bf16(tmem + (uint32_t)(ac * D), ad, bd, idesc, (term | ks) ? 1u : 0u);
      }
    tc::umma_commit(&pp.a_empty[st]);
    tc::umma_commit(&pp.acc_full[ac]);
    issued = it + 1;
  }
  // the last commit tracks every MMA issued before it
  if (issued > 0)
    mbar_wait_bounded(&pp.acc_full[(issued - 1) & 1], (uint32_t)(((issued - 1) / 2) & 1), 16u);
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A run of 32 coordinates with one beside a boundary, noted by the epilogue.
struct Again {
  uint8_t* out;                            // the run's codes in its page row
  int i;                                   // vector
  uint32_t row;                            // of the rotation table; run of the vector in bits 30, 31
};
// Noted per epilogue warp, in the warp's order; runs past that keep their first
// values.  At one run in 1,600 the 8 warps' lists last for 100,000 vectors of 128
// per SM and launch, 15 million in all; a vector beside a boundary that repeats fills
// them after 32 times.  (Redone at once in the epilogue, a run's
// cold code held up its warp: whole prompts 125 us against 107; by the locators
// between their tiles, it held up the tiles: 138 us.)
constexpr int kAgain = 32;

template <int D>
struct AppendSmem {
  static constexpr int OFF_B = 0;
  static constexpr int OFF_A = OFF_B + 2 * Shape<D>::kB;           // 2 stages of hi, lo
  static constexpr int OFF_BND = OFF_A + 4 * Shape<D>::kTerm;      // [256]
  static constexpr int OFF_W = OFF_BND + 1024;                     // [D] norm weights
  static constexpr int OFF_AGAIN = OFF_W + 4 * D;                  // noted runs, their counts
  static constexpr int OFF_REQ = OFF_AGAIN + AppendRoles<D>::kEpi * (kAgain * (int)sizeof(Again) + 4);
  static constexpr int OFF_VEC = OFF_REQ + kStagedBytes;           // [kRing]
  static constexpr int OFF_PIPE = OFF_VEC + kRing * (int)sizeof(Vecs);
  static constexpr int OFF_LUT = OFF_PIPE + kPipeBytes;
  static constexpr int LUT_BYTES = kSmem - 1024 - OFF_LUT;         // 1 KB: slack to align the base
  static_assert(LUT_BYTES >= 8 * 1024, "shared memory");
  static_assert(OFF_A % 1024 == 0 && Shape<D>::kTerm % 1024 == 0, "swizzled tiles");
  static_assert(OFF_VEC % 8 == 0 && OFF_PIPE % 8 == 0 && OFF_LUT % 16 == 0, "alignment");
};

// Four 16-bit values of a vector in fp32.
__device__ __forceinline__ void widen4(uint2 u, int dtype, float* v) {
  if (dtype == TQ_BF16) {
    v[0] = __uint_as_float(u.x << 16);
    v[1] = __uint_as_float(u.x & 0xFFFF0000u);
    v[2] = __uint_as_float(u.y << 16);
    v[3] = __uint_as_float(u.y & 0xFFFF0000u);
  } else {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
}

template <int N>
__device__ __forceinline__ float sum_lanes(float x) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The run's codes in 64 bits, a coordinate per lane; xs: D doubles of the warp's.
template <int D, int BITS, bool AXES>
__device__ __forceinline__ void exact_run(const RaggedTc& p, int which, const float* bnd,
                                          const Again& e, double* xs) {
  constexpr int nb = (1 << BITS) - 1;
  const int lane = threadIdx.x & 31;
  const HeadXform& f = p.f;
  const bool norm = which == 0 && f.weight;
  const int rot = which == 0 && f.cos_sin ? f.rot : 0, half = rot / 2;
  const int64_t* st = p.stride[which];
  const int n = p.by_h.div(e.i);
  const int64_t base = (int64_t)n * st[1] + (int64_t)(e.i - n * p.H) * st[0];
  const int64_t at_row = e.row & 0x3FFFFFFFu;
  auto value = [&](int d) {
    const double x = load_elem(p.x[which], p.dtype[which], base + d);
    return norm ? x * ((double)load_elem(f.weight, f.w_dtype, d) + f.w_offset) : x;
  };
  // the sums before the rotation (the head norm's) and of what it gives
  double raw = 0.0, ss = 0.0;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    const int d = lane + 32 * k;
    const double own = load_elem(p.x[which], p.dtype[which], base + d);
    raw += own * own;
    double x = value(d);
    if (d < rot) {
      const int a = f.interleaved ? d >> 1 : d < half ? d : d - half;    // angle
      const bool second = f.interleaved ? d & 1 : d >= half;
      const int with = f.interleaved ? d ^ 1 : second ? d - half : d + half;
      const int64_t row =
          AXES ? table_row(f, load_pos(p.pos, p.pos64, at_row * p.pos_stride +
                                                           f.axes.axis(a) * f.axes.stride), p.status)
               : at_row;
      const float* cs = f.cos_sin + row * rot;
      x = x * cs[a] + value(with) * (second ? cs[half + a] : -cs[half + a]);
    }
    ss += x * x;
    xs[d] = x;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    raw += __shfl_xor_sync(0xffffffffu, raw, o);
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  __syncwarp();
  const int col = 32 * (e.row >> 30) + lane;
  const float4* R = reinterpret_cast<const float4*>(
      p.rot + (which == 0 ? k_coord_at(col, D) : v_coord_at(col, D)) * D);
  double y[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
  for (int d = 0; d < D; d += 4) {
    const float4 w = __ldg(R + d / 4);
    y[0] += xs[d] * w.x;
    y[1] += xs[d + 1] * w.y;
    y[2] += xs[d + 2] * w.z;
    y[3] += xs[d + 3] * w.w;
  }
  __syncwarp();                            // before the next run's xs
  // the head norm's factor matters where the unit vector's floor of 1e-8 does
  const double r = norm ? rsqrt(raw / D + (double)f.eps) : 1.0;
  const double len = fmax(sqrt(ss) * r, 1e-8), v = ((y[0] + y[1]) + (y[2] + y[3])) * r;
  uint32_t code = 0;
  for (int k = 0; k < nb; ++k) code += bnd[k] * len < v;
#pragma unroll
  for (int x = 0; x < BITS; ++x) {
    const int sh = lane * BITS - 32 * x;   // the code's place in word x
    const uint32_t own = sh <= -BITS || sh >= 32 ? 0u : sh >= 0 ? code << sh : code >> -sh;
    const uint32_t word = __reduce_or_sync(0xffffffffu, own);
    if (lane == x) reinterpret_cast<uint32_t*>(e.out)[x] = word;
  }
}

// AXES: a rotation by several position axes (keys).
template <int D, int BITS, bool AXES>
__global__ void __launch_bounds__(AppendRoles<D>::kThreads, 1)
append_ragged_tc_kernel(const __grid_constant__ RaggedTc p, int which) {
  using S = Shape<D>;
  using W = AppendRoles<D>;
  constexpr int kMakers = W::kMakers, kThreads = W::kThreads;
  using SM = AppendSmem<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const Pipe pp = make_pipe(sm + SM::OFF_PIPE);
  float* lutpar = reinterpret_cast<float*>(sm + SM::OFF_PIPE + kPipeBytes - 16);
  float* bnd = reinterpret_cast<float*>(sm + SM::OFF_BND);
  Vecs* ring = reinterpret_cast<Vecs*>(sm + SM::OFF_VEC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nb = (1 << BITS) - 1;
  const int nvec = p.nvec;

  // the V kernel may start beside the K kernel (they share no byte); it ends
  // after it, so that whatever follows sees both
  pdl_launch_dependents();
  const OffsetCheck offsets(p.rv, tid);
  if (tid == 0) init_pipe(pp, kMakers, W::kEpi);
  if (warp == W::kIssuer) {
    tc::tmem_alloc(pp.tmem_slot, 2 * D);
    tc::tmem_relinquish();
  }
  for (int i = tid; i < nb; i += kThreads) bnd[i] = p.bnd[which][i];
  float* weight = reinterpret_cast<float*>(sm + SM::OFF_W);
  Again* again = reinterpret_cast<Again*>(sm + SM::OFF_AGAIN);    // [epilogue warps][kAgain]
  int* nagain = reinterpret_cast<int*>(again + W::kEpi * kAgain);
  if (which == 0 && p.f.weight)
    for (int i = tid; i < D; i += kThreads)
      weight[i] = load_elem(p.f.weight, p.f.w_dtype, i) + p.f.w_offset;
  const Requests requests = stage_requests(p.rv, sm + SM::OFF_REQ, tid, kThreads);
  stage_rotation<D, kThreads>(sm + SM::OFF_B, p.rot, which, tid);
  tc::fence_proxy_async_smem();
  tc::tc_fence_before();
  const bool run = !__syncthreads_or(offsets.fails(p.rv, tid, kThreads, p.status));
  // the locators need no more; the others agree on the lookup table
  const bool locator = warp >= W::kLocators && warp < W::kEpi0;
  auto others_sync = [&] {
    asm volatile("bar.sync 7, %0;" ::"n"(kThreads - 64) : "memory");
  };
  if (warp == 0) {
    float gap = 1.f;
    for (int i = lane; i + 1 < nb; i += 32) gap = fminf(gap, bnd[i + 1] - bnd[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) gap = fminf(gap, __shfl_xor_sync(0xffffffffu, gap, o));
    const float w = 0.4f * gap;
    const float span = fmaxf(fabsf(bnd[0]), fabsf(bnd[nb - 1]));
    const float L = ceilf(span / w) + 3.f, nc = 2.f * L + 1.f;
    const bool ok = w > 0.f && nc * 128.f <= (float)SM::LUT_BYTES && span < 1.f;
    if (lane == 0) {
      lutpar[0] = 1.f / (2.f * L * w);     // u = sat(v * lutpar[0] + 0.5)
      lutpar[1] = 2.f * L;                 // cell = round(u * 2L)
      lutpar[2] = ok ? nc : 0.f;
      lutpar[3] = w;
    }
  }
  if (!locator) others_sync();
  const int ncells = locator ? 0 : (int)lutpar[2];
  if (!locator) {
    const float w = lutpar[3], L = 0.5f * lutpar[1];
    for (int i = tid < 32 * W::kLocators ? tid : tid - 64; i < ncells * 16; i += kThreads - 64) {
      const int c = i >> 4;
      const float wl = ((float)c - L - 1.f) * w, wh = ((float)c - L + 1.f) * w;
      const int base = bucketize_lt(bnd, nb, wl);
      const float nbk = (base < nb && bnd[base] <= wh) ? -bnd[base] * kCmp : -INFINITY;
      reinterpret_cast<float2*>(sm + SM::OFF_LUT)[i] = make_float2(nbk, (float)base);
    }
    tc::fence_proxy_async_smem();
    tc::tc_fence_before();
    others_sync();
    tc::tc_fence_after();
  }
  const uint32_t tmem = *pp.tmem_slot;
  const int first = run ? blockIdx.x : p.ntiles, step = gridDim.x;
  const bool use_lo = p.use_lo[which] != 0;

  if (warp < kMakers) {
    // ------------------------------------------------------------ operand makers
    // D / 16 lanes per vector, two groups of eight dims each
    constexpr int LV = D / 16, RPI = 32 / LV, NIT = W::kVecs / RPI;   // vectors per pass, passes
    static_assert(NIT >= 1, "a warp's vectors fill its lanes");
    const int l = lane % LV, sub = lane / LV;
    const HeadXform f = which == 0 ? p.f : HeadXform{};
    // the groups: partners of the rotation (halves), or plain halves of the vector
    const int half = f.rot / 2;
    const bool pairs = f.cos_sin && !f.interleaved;        // (i, half + i)
    int ga = 8 * l, gb = D / 2 + 8 * l;
    bool turn = f.cos_sin != nullptr;                      // this lane rotates
    if (pairs) {
      if (ga < half) { gb = half + ga; }
      else { ga = f.rot + 2 * (8 * l - half); gb = ga + 8; turn = false; }
    }
    const bool turn_a = turn && (pairs || ga < f.rot), turn_b = turn && !pairs && gb < f.rot;
    const int64_t* xs = p.stride[which];
    const int dtype = p.dtype[which];
    const bool wide = dtype == TQ_F32;
    // 16-bit values of a tile's vectors (32-bit ones would take twice the
    // registers: loaded when they are used)
    struct Raw { uint4 a[NIT], b[NIT]; };
    auto base_of = [&](int i) {
      const int n = p.by_h.div(i);
      return (int64_t)n * xs[1] + (int64_t)(i - n * p.H) * xs[0];
    };
    auto load_raw = [&](Raw& x, int v0) {
#pragma unroll
      for (int k = 0; k < NIT; ++k) {
        const int i = v0 + k * RPI + sub;
        x.a[k] = x.b[k] = make_uint4(0u, 0u, 0u, 0u);
        if (!wide && i < nvec) {
          const uint16_t* at = static_cast<const uint16_t*>(p.x[which]) + base_of(i);
          x.a[k] = __ldg(reinterpret_cast<const uint4*>(at + ga));
          x.b[k] = __ldg(reinterpret_cast<const uint4*>(at + gb));
        }
      }
    };
    auto vec0 = [&](int tile) { return tile * kM + W::kVecs * warp; };
    auto axis_row = [&](int64_t n, int a) {
      return table_row(p.f, load_pos(p.pos, p.pos64, n * p.pos_stride + a * p.f.axes.stride), p.status);
    };
    Raw cur, nxt;
    if (first < p.ntiles) load_raw(cur, vec0(first));
    int it = 0;
    for (int tile = first; tile < p.ntiles; tile += step, ++it) {
      const int st = it & 1;
      const int v0 = vec0(tile);
      if (tile + step < p.ntiles) load_raw(nxt, vec0(tile + step));
      bool ok = true;
      if (it == 0 || f.cos_sin == nullptr)
        ok = wait_for(&pp.loc_full[it % kRing], (uint32_t)((it / kRing) & 1), pp.abort_flag, p.status);
      if (f.cos_sin && ok && tile + step < p.ntiles) {
        // the next tile's rows of the rotation table on their way into L1
        const int e = (it + 1) % kRing;
        ok = wait_for(&pp.loc_full[e], (uint32_t)(((it + 1) / kRing) & 1), pp.abort_flag, p.status);
        constexpr int LINES = 32 / W::kVecs;               // 128-byte lines per lane's vector
        const int64_t to = ring[e].row[W::kVecs * warp + lane / LINES];
        for (int a = 0; a < (AXES ? p.f.axes.n : 1); ++a) {
          int64_t row = to;
          if constexpr (AXES) {                            // a row that the table has not is flagged where it turns
            if (to < 0) break;
            row = load_pos(p.pos, p.pos64, to * p.pos_stride + a * p.f.axes.stride);
            if ((uint64_t)row >= (uint64_t)f.positions) continue;
          }
          const float* at = f.cos_sin + row * f.rot;
          for (int c = 32 * (lane % LINES); c < f.rot; c += 32 * LINES)
            asm volatile("prefetch.global.L1 [%0];" ::"l"(at + c));
        }
      }
      ok = ok && (it < 2 || wait_for(&pp.a_empty[st], (uint32_t)(((it / 2) - 1) & 1),
                                     pp.abort_flag, p.status));
      if (!__all_sync(0xffffffffu, ok)) break;
      Vecs& vec = ring[it % kRing];
      // AXES: the angles of a token serve its heads, which lie next to each other
      int64_t turned = -1;
      float ac[8], as[8];
      unsigned char* hi = sm + SM::OFF_A + st * 2 * S::kTerm;
#pragma unroll
      for (int k = 0; k < NIT; ++k) {
        const int vi = k * RPI + sub;                      // vector of the warp's
        float v[16];
        if (wide) {
          const bool in = v0 + vi < nvec;
          const float* x = static_cast<const float*>(p.x[which]) + base_of(in ? v0 + vi : 0);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 y = __ldg(reinterpret_cast<const float4*>(x + (e < 8 ? ga + e : gb + e - 8)));
            v[e] = in ? y.x : 0.f;
            v[e + 1] = in ? y.y : 0.f;
            v[e + 2] = in ? y.z : 0.f;
            v[e + 3] = in ? y.w : 0.f;
          }
        } else {
          widen4(make_uint2(cur.a[k].x, cur.a[k].y), dtype, v);
          widen4(make_uint2(cur.a[k].z, cur.a[k].w), dtype, v + 4);
          widen4(make_uint2(cur.b[k].x, cur.b[k].y), dtype, v + 8);
          widen4(make_uint2(cur.b[k].z, cur.b[k].w), dtype, v + 12);
        }
        if (f.weight) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss = fmaf(v[e], v[e], ss);
          const float r = rsqrtf(fmaf(sum_lanes<LV>(ss), 1.f / (float)D, f.eps));
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 w = *reinterpret_cast<const float4*>(weight + (e < 8 ? ga + e : gb + e - 8));
            v[e] *= r * w.x;
            v[e + 1] *= r * w.y;
            v[e + 2] *= r * w.z;
            v[e + 3] *= r * w.w;
          }
        }
        if (f.cos_sin) {
          const int64_t to = vec.row[W::kVecs * warp + vi];
          const float* cs = f.cos_sin + (AXES ? 0 : to * f.rot);
          auto rotate = [](float& a, float& b, float c, float s) {
            const float t = a * c - b * s;
            b = b * c + a * s;
            a = t;
          };
          if constexpr (AXES) {
            auto row_of = [&](int a) { return axis_row(to, a); };
            if (to >= 0 && to != turned) {                 // without a place: as it is, nobody reads it
              turned = to;
              if (pairs) {
                if (turn_a) load_axes<8>(ac, as, p.f, ga, row_of);
              } else {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                  if (!(g ? turn_b : turn_a)) continue;
                  float c4[4], s4[4];
                  load_axes<4>(c4, s4, p.f, (g ? gb : ga) / 2, row_of);
#pragma unroll
                  for (int e = 0; e < 4; ++e) { ac[4 * g + e] = c4[e]; as[4 * g + e] = s4[e]; }
                }
              }
            }
            if (pairs) {
              if (turn_a && to >= 0)
#pragma unroll
                for (int e = 0; e < 8; ++e) rotate(v[e], v[8 + e], ac[e], as[e]);
            } else {
#pragma unroll
              for (int g = 0; g < 2; ++g)
                if ((g ? turn_b : turn_a) && to >= 0)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    rotate(v[8 * g + 2 * e], v[8 * g + 2 * e + 1], ac[4 * g + e], as[4 * g + e]);
            }
          } else if (pairs) {
            if (turn_a) {
#pragma unroll
              for (int e = 0; e < 8; e += 4) {
                const float4 c = __ldg(reinterpret_cast<const float4*>(cs + ga + e));
                const float4 s = __ldg(reinterpret_cast<const float4*>(cs + half + ga + e));
                rotate(v[e], v[8 + e], c.x, s.x);
                rotate(v[e + 1], v[9 + e], c.y, s.y);
                rotate(v[e + 2], v[10 + e], c.z, s.z);
                rotate(v[e + 3], v[11 + e], c.w, s.w);
              }
            }
          } else {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (g ? turn_b : turn_a) {
                const int at = (g ? gb : ga) / 2;
                const float4 c = __ldg(reinterpret_cast<const float4*>(cs + at));
                const float4 s = __ldg(reinterpret_cast<const float4*>(cs + half + at));
                rotate(v[8 * g], v[8 * g + 1], c.x, s.x);
                rotate(v[8 * g + 2], v[8 * g + 3], c.y, s.y);
                rotate(v[8 * g + 4], v[8 * g + 5], c.z, s.z);
                rotate(v[8 * g + 6], v[8 * g + 7], c.w, s.w);
              }
            }
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss = fmaf(v[e], v[e], ss);
        ss = sum_lanes<LV>(ss);
        // the norm and its reciprocal from one rsqrt (2^-22), s = 2^(10 -
        // exponent of the norm) from 2^-118 to 2^100 and its reciprocal from
        // the exponent bits: no division or root on the way
        const float rn = rsqrtf(ss);
        const float n = ss == 0.f || ss == INFINITY ? ss : ss * rn;
        const int ex = max((int)((__float_as_uint(n) >> 23) & 255u) - 127, -90);
        const float s = __uint_as_float((uint32_t)(127 + 10 - ex) << 23);
        const float rs = __uint_as_float((uint32_t)(127 - 10 + tmin(ex, 127)) << 23);
        const int r = W::kVecs * warp + vi;
        if (l == 0) {
          vec.n[r] = n;
          vec.inv[r] = (n < 1e-8f ? 1e8f : rn) * rs * (1.f / kRScale);
        }
        const uint32_t aa = chunk_at<kM>(r, ga >> 3), ab = chunk_at<kM>(r, gb >> 3);
        uint32_t h[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_pair(v[2 * e] * s, v[2 * e + 1] * s, h[e], lo[e]);
        *reinterpret_cast<uint4*>(hi + aa) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(hi + ab) = make_uint4(h[4], h[5], h[6], h[7]);
        if (use_lo) {
          *reinterpret_cast<uint4*>(hi + S::kTerm + aa) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<uint4*>(hi + S::kTerm + ab) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        }
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_cta(&pp.a_full[st]);
      cur = nxt;
    }
  } else if (warp == W::kIssuer) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t a0 = smem_u32(sm + SM::OFF_A), b0 = smem_u32(sm + SM::OFF_B);
      issue_tiles<D, 2, false>(pp, tmem, first, step, p.ntiles, p.status,
                               [&](int st, int term, uint32_t& a, uint32_t& b) {
                                 a = a0 + st * 2 * S::kTerm + (term == 2 ? S::kTerm : 0);
                                 b = b0 + (term == 1 ? S::kB : 0);
                                 return term < (use_lo ? 3 : 2);
                               });
    }
    __syncwarp();
  } else if (warp < W::kEpi0) {
    locate_tiles<AXES>(p, pp, ring, requests, warp - W::kLocators, first, step);
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int NCH = D / W::kSplit / 32;                // runs of 32 columns per thread
    const int q = warp & 3, part = (warp - W::kEpi0) >> 2;
    const int r = 32 * q + lane;
    const int row_bytes = D * BITS / 8;
    const int sec = which == 0 ? p.g.off_k : p.g.off_v, noff = which == 0 ? p.g.off_kn : p.g.off_vn;
    const uint32_t lane_off = smem_u32(sm + SM::OFF_LUT) + (uint32_t)((lane & 15) * 8) -
                              (0x4B000000u << 7);
    const float par0 = lutpar[0], c2l = lutpar[1];
    Again* mine = again + kAgain * (warp - W::kEpi0);
    int it = 0, noted = 0;
    for (int tile = first; tile < p.ntiles; tile += step, ++it) {
      const int ac = it & 1;
      bool ok = wait_for(&pp.acc_full[ac], (uint32_t)((it / 2) & 1), pp.abort_flag, p.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc::tc_fence_after();
      const Vecs& vec = ring[it % kRing];
      uint8_t* const page = vec.page[r];
      const int slot = vec.slot[r];
      const float n = vec.n[r], inv = vec.inv[r], ca = inv * par0, cK = inv * kCmp;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        const int run = part * NCH + ch;                   // 32 positions of the row
        uint32_t yb[32];
        tc::tmem_ld_x32(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(ac * D + 32 * run), yb);
        tc::tmem_wait_ld();
        if (ch == NCH - 1) {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cta(&pp.acc_empty[ac]);
        }
        uint32_t words[BITS];
#pragma unroll
        for (int x = 0; x < BITS; ++x) words[x] = 0u;
        float near = INFINITY;             // least distance to a boundary, times 2^100
        if (ncells > 0) {
          // codes gather in runs of <= 23 bits as acc = 2^23 + field, exactly
          auto flush = [&](float acc, int o, int len) {
            const uint32_t bits = __float_as_uint(acc) & ((1u << len) - 1u);
            const int wi = o >> 5, sh = o & 31;
            words[wi] += bits << sh;
            if (sh + len > 32) words[wi + 1] += bits >> (32 - sh);
          };
          float acc = 8388608.f;
          int gs = 0, gl = 0;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int bo = j * BITS;
            if (gl > 0 && (gl + BITS > 23 || (bo & 31) == 0)) {
              flush(acc, gs, gl);
              acc = 8388608.f;
              gs = bo;
              gl = 0;
            }
            const float y = __uint_as_float(yb[j]);
            const float u = __saturatef(fmaf(y, ca, 0.5f));
            const float cell = fmaf(u, c2l, 8388608.f);
            const float2 e = tc::lds_f2((__float_as_uint(cell) << 7) + lane_off);
            const float over = fmaf(y, cK, e.x);
            const float above = __saturatef(over * kCmp);
            near = fminf(near, fabsf(over));
            acc = fmaf(e.y + above, (float)(1u << gl), acc);
            gl += BITS;
          }
          flush(acc, gs, gl);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float y = __uint_as_float(yb[j]) * inv;
            const uint32_t code = (uint32_t)bucketize_lt(bnd, nb, y);
            near = fminf(near, kCmp * fminf(code > 0 ? fabsf(y - bnd[code - 1]) : 1.f,
                                            code < nb ? fabsf(y - bnd[code]) : 1.f));
            const int bo = j * BITS, wi = bo >> 5, sh = bo & 31;
            words[wi] += code << sh;
            if (sh + BITS > 32) words[wi + 1] += code >> (32 - sh);
          }
        }
        if (page) {
          uint8_t* row = page + sec + slot * row_bytes + run * (4 * BITS);
          if constexpr (BITS % 4 == 0) {
#pragma unroll
            for (int x = 0; x < BITS / 4; ++x)
              reinterpret_cast<uint4*>(row)[x] = make_uint4(words[4 * x], words[4 * x + 1],
                                                            words[4 * x + 2], words[4 * x + 3]);
          } else if constexpr (BITS % 2 == 0) {
#pragma unroll
            for (int x = 0; x < BITS / 2; ++x)
              reinterpret_cast<uint2*>(row)[x] = make_uint2(words[2 * x], words[2 * x + 1]);
          } else {
#pragma unroll
            for (int x = 0; x < BITS; ++x) reinterpret_cast<uint32_t*>(row)[x] = words[x];
          }
        }
        const bool note = near < kNear * kCmp && n > 0.f && page;
        const uint32_t notes = __ballot_sync(0xffffffffu, note);
        if (notes) {
          const int at = noted + __popc(notes & ((1u << lane) - 1u));
          if (note && at < kAgain)
            mine[at] = {page + sec + slot * row_bytes + run * (4 * BITS), tile * kM + r,
                        (uint32_t)vec.row[r] | (uint32_t)run << 30};
          noted += __popc(notes);
        }
      }
      if (page && part == 0)
        reinterpret_cast<__half*>(page + noff)[slot] = __float2half_rn(n);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_cta(&pp.loc_free[it % kRing]);
    }
    if (lane == 0) nagain[warp - W::kEpi0] = tmin(noted, kAgain);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == W::kIssuer) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 2 * D);
  }
  // runs beside a boundary again, over the operands' place
  double* xs = reinterpret_cast<double*>(sm + SM::OFF_A) + D * warp;
  for (int w = 0, k = warp; w < W::kEpi; ++w) {
    for (; k < nagain[w]; k += kThreads / 32)
      exact_run<D, BITS, AXES>(p, which, bnd, again[kAgain * w + k], xs);
    k -= nagain[w];
  }
  pdl_wait();
}

// ---------------------------------------------------------------------------
// read-back
// ---------------------------------------------------------------------------
// LO: c as hi + lo (fp16 and fp32 results), one operand stage; else c = hi, two.
template <int D, int BITS, bool LO>
struct ReadSmem {
  static constexpr int STAGES = LO ? 1 : 2;
  static constexpr bool kPair = BITS <= 4;                         // table of code pairs
  using Chunk = typename std::conditional<(BITS <= 4), uint32_t, uint64_t>::type;   // 8 codes
  // entry: fp16 pair hi (and lo) of two codes, or one code's {hi, lo}; copies
  // for 32 lanes of 4-byte entries, 16 of 8-byte ones: 128 bytes
  static constexpr int OFF_B = 0;
  static constexpr int OFF_A = OFF_B + 2 * Shape<D>::kB;
  // results on their way out, [rows][D]: all 128 rows of 16-bit values; of 32-bit
  // ones half a tile at a time
  static constexpr int OFF_OUT = OFF_A + (LO ? 2 : STAGES) * Shape<D>::kTerm;
  static constexpr int OFF_LUT = OFF_OUT + kM * D * 2;
  static constexpr int LUT_BYTES = (1 << (kPair ? 2 * BITS : BITS)) * 128;
  static constexpr int OFF_REQ = OFF_LUT + LUT_BYTES;              // offsets and lengths
  static constexpr int OFF_VEC = OFF_REQ + kStagedBytes;           // [kRing]
  static constexpr int OFF_PIPE = OFF_VEC + kRing * (int)sizeof(Vecs);
  static constexpr int BYTES = OFF_PIPE + kPipeBytes + 1024;
  static_assert(BYTES <= kSmem, "shared memory");
};

// The 8 codes of chunk c of a packed row: 8 * BITS bits from byte c * BITS on.
template <int BITS>
__device__ __forceinline__ uint64_t load_chunk(const uint8_t* row, int c) {
  const int off = c * BITS;
  if constexpr (BITS == 8) return __ldg(reinterpret_cast<const unsigned long long*>(row + off));
  if constexpr (BITS == 4) return __ldg(reinterpret_cast<const uint32_t*>(row + off));
  if constexpr (BITS == 2) return __ldg(reinterpret_cast<const uint16_t*>(row + off));
  if constexpr (BITS == 1) return __ldg(row + off);
  // the words that hold them (reads stay inside the page: norms follow the codes)
  const uint32_t* w = reinterpret_cast<const uint32_t*>(row + (off & ~3));
  const int sh = (off & 3) * 8;
  uint64_t v = (uint64_t)__ldg(w) | ((uint64_t)__ldg(w + 1) << 32);
  v >>= sh;
  if (BITS > 5 && sh > 0) v |= (uint64_t)__ldg(w + 2) << (64 - sh);
  return v;
}

template <int D, int BITS, bool LO>
__global__ void __launch_bounds__(ReadRoles<D>::kThreads, 1)
read_ragged_tc_kernel(RaggedTc p, int which) {
  using S = Shape<D>;
  using W = ReadRoles<D>;
  constexpr int kMakers = W::kMakers, kThreads = W::kThreads;
  using SM = ReadSmem<D, BITS, LO>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const Pipe pp = make_pipe(sm + SM::OFF_PIPE);
  Vecs* ring = reinterpret_cast<Vecs*>(sm + SM::OFF_VEC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nvec = p.nvec;

  // the V kernel may start beside the K kernel (they share no byte); it ends
  // after it, so that whatever follows sees both
  pdl_launch_dependents();
  const OffsetCheck offsets(p.rv, tid);
  if (tid == 0) init_pipe(pp, kMakers, W::kEpi);
  if (warp == W::kIssuer) {
    tc::tmem_alloc(pp.tmem_slot, 2 * D);
    tc::tmem_relinquish();
  }
  const Requests requests = stage_requests(p.rv, sm + SM::OFF_REQ, tid, kThreads);
  stage_rotation<D, kThreads>(sm + SM::OFF_B, p.rot, which, tid);
  {
    const float* cent = p.cent[which];
    constexpr uint32_t mask = (1u << BITS) - 1u;
    for (int i = tid; i < SM::LUT_BYTES / 16; i += kThreads) {
      const uint32_t e = (uint32_t)i >> 3;
      uint32_t h, l;
      if (SM::kPair) {
        split_pair(__ldg(cent + (e & mask)), __ldg(cent + (e >> BITS)), h, l);
      } else {
        split_pair(__ldg(cent + e), 0.f, h, l);            // low halves: hi, lo of one code
        h = (h & 0xFFFFu) | (l << 16);
      }
      const uint4 x = SM::kPair && LO ? make_uint4(h, l, h, l) : make_uint4(h, h, h, h);
      reinterpret_cast<uint4*>(sm + SM::OFF_LUT)[i] = x;
    }
  }
  tc::fence_proxy_async_smem();
  tc::tc_fence_before();
  const bool run = !__syncthreads_or(offsets.fails(p.rv, tid, kThreads, p.status));
  tc::tc_fence_after();
  const uint32_t tmem = *pp.tmem_slot;
  const int first = run ? blockIdx.x : p.ntiles, step = gridDim.x;
  const int row_bytes = D * BITS / 8;
  const int sec = which == 0 ? p.g.off_k : p.g.off_v, noff = which == 0 ? p.g.off_kn : p.g.off_vn;

  if (warp < kMakers) {
    // ------------------------------------------------------------ operand makers
    // D / 8 lanes per vector, eight codes each
    constexpr int LV = D / 8, RPI = 32 / LV, NIT = W::kVecs / RPI;
    const int l = lane % LV, sub = lane / LV;
    const unsigned char* lut = sm + SM::OFF_LUT + (SM::kPair && LO ? 8 * (lane & 15) : 4 * lane);
    using Chunk = typename SM::Chunk;
    struct Raw { Chunk codes[NIT]; float n; };
    // a tile's codes and (lanes < kVecs) norms, once its places are known
    auto load_raw = [&](Raw& x, int it) -> bool {
      if (!__all_sync(0xffffffffu, wait_for(&pp.loc_full[it % kRing], (uint32_t)((it / kRing) & 1),
                                            pp.abort_flag, p.status)))
        return false;
      const Vecs& vec = ring[it % kRing];
      const int r0 = W::kVecs * warp;
#pragma unroll
      for (int k = 0; k < NIT; ++k) {
        const int r = r0 + k * RPI + sub;
        const uint8_t* page = vec.page[r];
        x.codes[k] = page ? (Chunk)load_chunk<BITS>(page + sec + vec.slot[r] * row_bytes, l) : (Chunk)0;
      }
      x.n = 0.f;
      if (lane < W::kVecs && vec.page[r0 + lane])
        x.n = __half2float(__ldg(reinterpret_cast<const __half*>(vec.page[r0 + lane] + noff) +
                                 vec.slot[r0 + lane]));
      return true;
    };
    Raw cur, nxt;
    bool more = first < p.ntiles && load_raw(cur, 0);
    int it = 0;
    for (int tile = first; more && tile < p.ntiles; tile += step, ++it) {
      const int st = it % SM::STAGES;
      if (tile + step < p.ntiles) more = load_raw(nxt, it + 1);
      bool ok = it < SM::STAGES ||
                wait_for(&pp.a_empty[st], (uint32_t)(((it / SM::STAGES) - 1) & 1), pp.abort_flag,
                         p.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane < W::kVecs) ring[it % kRing].n[W::kVecs * warp + lane] = cur.n;
      unsigned char* hi = sm + SM::OFF_A + st * S::kTerm;
#pragma unroll
      for (int k = 0; k < NIT; ++k) {
        const Chunk codes = cur.codes[k];
        const int r = W::kVecs * warp + k * RPI + sub;
        uint32_t h[4], lo[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (SM::kPair) {
            const uint32_t idx = (uint32_t)(codes >> (2 * BITS * e)) & ((1u << (2 * BITS)) - 1u);
            if constexpr (LO) {
              const uint2 x = *reinterpret_cast<const uint2*>(lut + idx * 128);
              h[e] = x.x;
              lo[e] = x.y;
            } else {
              h[e] = *reinterpret_cast<const uint32_t*>(lut + idx * 128);
            }
          } else {
            const uint32_t i0 = (uint32_t)(codes >> (2 * BITS * e)) & ((1u << BITS) - 1u);
            const uint32_t i1 = (uint32_t)(codes >> (2 * BITS * e + BITS)) & ((1u << BITS) - 1u);
            const uint32_t a = *reinterpret_cast<const uint32_t*>(lut + i0 * 128);
            const uint32_t b = *reinterpret_cast<const uint32_t*>(lut + i1 * 128);
            h[e] = __byte_perm(a, b, 0x5410);
            lo[e] = __byte_perm(a, b, 0x7632);
          }
        }
        const uint32_t at = chunk_at<kM>(r, l);
        *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
        if (LO)
          *reinterpret_cast<uint4*>(hi + S::kTerm + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_cta(&pp.a_full[st]);
      cur = nxt;
    }
  } else if (warp == W::kIssuer) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t a0 = smem_u32(sm + SM::OFF_A), b0 = smem_u32(sm + SM::OFF_B);
      issue_tiles<D, SM::STAGES, true>(pp, tmem, first, step, p.ntiles, p.status,
                                       [&](int st, int term, uint32_t& a, uint32_t& b) {
                                         a = a0 + st * S::kTerm + (term == 2 ? S::kTerm : 0);
                                         b = b0 + (term == 1 ? S::kB : 0);
                                         return term < (LO ? 3 : 2);
                                       });
    }
    __syncwarp();
  } else if (warp < W::kEpi0) {
    locate_tiles<false>(p, pp, ring, requests, warp - W::kLocators, first, step);
  } else {
    // ------------------------------------------------------------ epilogue
    // The kSplit warps of a lane quarter hold 32 rows x 32 columns each; they
    // put them into shared memory and take ROWS whole rows each out of it.
    constexpr int ROWS = 32 / W::kSplit;
    const int q = warp & 3, part = (warp - W::kEpi0) >> 2;
    const int es = p.dtype[which] == TQ_F32 ? 4 : 2;
    const bool bf16 = p.dtype[which] == TQ_BF16;
    const int64_t* xs = p.stride[which];
    char* const dst = static_cast<char*>(const_cast<void*>(p.x[which]));
    unsigned char* out = sm + SM::OFF_OUT + q * (32 * D * 2);
    // 16-byte piece c of the quarter's row r (16-bit values), moved so that a
    // warp's pieces spread over the banks
    constexpr int PIECES = D / 8;
    auto piece = [&](int r, int c) { return out + (r * PIECES + (c ^ (r & 7))) * 16; };
    auto quarter_sync = [&] {
      asm volatile("bar.sync %0, %1;" ::"r"(1 + q), "r"(32 * W::kSplit) : "memory");
    };
    int it = 0;
    for (int tile = first; tile < p.ntiles; tile += step, ++it) {
      const int ac = it & 1;
      uint32_t all = wait_for(&pp.acc_full[ac], (uint32_t)((it / 2) & 1), pp.abort_flag, p.status);
      // the lane quarter's warps go on or leave together (and: the rows of the
      // last tile have left shared memory)
      asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %0, 0;\n"
                   " bar.red.and.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
                   : "+r"(all) : "r"(1 + q), "r"(32 * W::kSplit) : "memory");
      if (!all) {
        *pp.abort_flag = 1;
        break;
      }
      tc::tc_fence_after();
      uint32_t x[32];
      tc::tmem_ld_x32(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(ac * D + 32 * part), x);
      const Vecs& vec = ring[it % kRing];
      const float n = vec.n[32 * q + lane] * (1.f / kRScale);
      // lane < ROWS: the offset of the row it sends out, and what becomes of it
      const int mine = 32 * q + ROWS * part + lane, v = tile * kM + mine;
      int state = 0;
      int64_t at = 0;
      if (lane < ROWS && v < nvec) {
        state = vec.state[mine];
        const int row = p.by_h.div(v);
        at = ((int64_t)row * xs[1] + (int64_t)(v - row * p.H) * xs[0]) * es;
      }
      tc::tmem_wait_ld();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive_cta(&pp.acc_empty[ac]);
        tc::mbar_arrive_cta(&pp.loc_free[it % kRing]);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * n);
      if (es == 2) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = __uint_as_float(x[8 * c + 2 * e]), b = __uint_as_float(x[8 * c + 2 * e + 1]);
            const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
            h[e] = bf16 ? *reinterpret_cast<const uint32_t*>(&y) : pack_half2(a, b);
          }
          *reinterpret_cast<uint4*>(piece(lane, 4 * part + c)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        quarter_sync();
        if (p.vec[which]) {
#pragma unroll
          for (int i = 0; i < ROWS * PIECES / 32; ++i) {
            const int rr = (32 * i + lane) / PIECES, c = lane % PIECES;
            const int64_t o = __shfl_sync(0xffffffffu, at, rr);
            const int stt = __shfl_sync(0xffffffffu, state, rr);
            uint4 y = *reinterpret_cast<const uint4*>(piece(ROWS * part + rr, c));
            if (stt == 1) y = make_uint4(0, 0, 0, 0);
            if (stt) *reinterpret_cast<uint4*>(dst + o + 16 * c) = y;
          }
        } else {
          for (int i = lane; i < ROWS * D; i += 32) {
            const int rr = i / D, d = i % D;
            const int64_t o = __shfl_sync(0xffffffffu, at, rr);
            const int stt = __shfl_sync(0xffffffffu, state, rr);
            const uint16_t y = reinterpret_cast<const uint16_t*>(piece(ROWS * part + rr, d / 8))[d % 8];
            if (stt) *reinterpret_cast<uint16_t*>(dst + o + 2 * d * xs[2]) = stt == 1 ? (uint16_t)0 : y;
          }
        }
      } else {
        // 32-bit values: the even, then the odd rows of the quarter
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          if (odd) quarter_sync();
          if ((lane & 1) == odd) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(out + (lane & ~1) * PIECES * 16 +
                                        (((8 * part + c) ^ ((lane >> 1) & 7)) << 4)) =
                  make_uint4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
          }
          quarter_sync();
          for (int i = lane; i < ROWS / 2 * D; i += 32) {
            const int pr = i / D, d = i % D, rr = 2 * pr + odd;   // row of this warp's ROWS
            const int row = ROWS * part + 2 * pr;                 // even row of the quarter
            const int64_t o = __shfl_sync(0xffffffffu, at, rr);
            const int stt = __shfl_sync(0xffffffffu, state, rr);
            const uint32_t y = reinterpret_cast<const uint32_t*>(
                out + row * PIECES * 16 + (((d / 4) ^ ((row >> 1) & 7)) << 4))[d % 4];
            if (stt) *reinterpret_cast<uint32_t*>(dst + o + 4 * d * xs[2]) = stt == 1 ? 0u : y;
          }
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == W::kIssuer) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 2 * D);
  }
  pdl_wait();
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
using RaggedFn = void (*)(RaggedTc, int);

template <int D, bool AXES>
RaggedFn append_fn(int bits) {
  switch (bits) {
    case 1: return append_ragged_tc_kernel<D, 1, AXES>;
    case 2: return append_ragged_tc_kernel<D, 2, AXES>;
    case 3: return append_ragged_tc_kernel<D, 3, AXES>;
    case 4: return append_ragged_tc_kernel<D, 4, AXES>;
    case 5: return append_ragged_tc_kernel<D, 5, AXES>;
    case 6: return append_ragged_tc_kernel<D, 6, AXES>;
    case 7: return append_ragged_tc_kernel<D, 7, AXES>;
    default: return append_ragged_tc_kernel<D, 8, AXES>;
  }
}

template <int D, bool LO>
RaggedFn read_fn(int bits, int& bytes) {
#define TQ_RD(B) case B: bytes = ReadSmem<D, B, LO>::BYTES; return read_ragged_tc_kernel<D, B, LO>;
  switch (bits) { TQ_RD(1) TQ_RD(2) TQ_RD(3) TQ_RD(4) TQ_RD(5) TQ_RD(6) TQ_RD(7) TQ_RD(8) }
#undef TQ_RD
  return nullptr;
}

RaggedTc tc_params(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                   const tq_tensor4* const x[2], const tq_ragged* batch, uint32_t* status) {
  RaggedTc p = {};
  p.g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.cent[0] = t->k_centroids; p.cent[1] = t->v_centroids;
  p.bnd[0] = t->k_boundaries; p.bnd[1] = t->v_boundaries;
  p.rot = t->rot;
  p.pages = c->pages;
  p.pm = page_map(c);
  p.status = status;
  for (int w = 0; w < 2; ++w) {
    if (!x[w]) continue;
    p.x[w] = x[w]->data;
    p.dtype[w] = x[w]->dtype;
    for (int i = 0; i < 3; ++i) p.stride[w][i] = x[w]->stride[i + 1];
    p.H = (int)x[w]->shape[1];
    p.rv = ragged_view(batch, x[w]->shape[2], c);
  }
  p.nvec = (int)(p.rv.N * p.H);
  p.by_h = fast_div(p.H);
  p.ntiles = (p.nvec + kM - 1) / kM;
  return p;
}

// `beside`: may start before the previous launch (the K kernel) has ended.
int launch_one(RaggedFn fn, unsigned grid, int threads, int bytes, cudaStream_t st,
               const RaggedTc& p, int which, bool beside, const char* what) {
  if (beside) return launch_result(launch_pdl(fn, dim3(grid), dim3(threads), bytes, st, p, which), what);
  fn<<<grid, threads, bytes, st>>>(p, which);
  return check_launch(what);
}

// Rows that take 16-byte loads and stores.
bool rows_aligned(const tq_tensor4* x) {
  const int es = x->dtype == TQ_F32 ? 4 : 2;
  if (x->stride[3] != 1 || reinterpret_cast<uintptr_t>(x->data) % 16) return false;
  for (int i = 1; i < 3; ++i)
    if (x->shape[i] > 1 && (x->stride[i] * es) % 16) return false;
  return true;
}

}  // namespace

// Both return TQ_OK when they ran, 1 when they do not apply, or an error.
int launch_append_ragged_tc(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                            const tq_tensor4* k, const tq_tensor4* v, const tq_ragged* batch,
                            const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm,
                            const tq_positions* pos, uint32_t* status, cudaStream_t st) {
  const int D = G->head_dim;
  if (D != 64 && D != 128) return 1;
  if (k->shape[1] * k->shape[2] > INT32_MAX - kM || (rope && (rope->rot_dim % 16 || rope->positions >> 30))) return 1;
  if (axes && k->shape[2] >> 30) return 1;                 // a noted run holds 30 bits of its row
  if (reinterpret_cast<uintptr_t>(t->rot) % 16) return 1;
  const tq_tensor4* x[2] = {k, v};
  for (int w = 0; w < 2; ++w)
    if (!rows_aligned(x[w])) return 1;
  RaggedTc p = tc_params(G, t, c, x, batch, status);
  p.f = head_xform(rope, axes, norm);
  p.pos = pos ? pos->data : nullptr;
  p.pos64 = pos && pos->bits == 64;
  p.pos_stride = pos ? pos->stride[1] : 0;
  p.use_lo[0] = rope || norm || k->dtype == TQ_F32;
  p.use_lo[1] = v->dtype == TQ_F32;
  const unsigned grid = (unsigned)tmin(p.ntiles, device_sm_count());
  for (int w = 0; w < 2; ++w) {
    const int bits = w == 0 ? G->key_bits : G->value_bits;
    const bool many = w == 0 && p.f.axes.n > 0;
    RaggedFn fn = D == 128 ? (many ? append_fn<128, true>(bits) : append_fn<128, false>(bits))
                           : (many ? append_fn<64, true>(bits) : append_fn<64, false>(bits));
    if (set_smem_attr((const void*)fn, kSmem) != TQ_OK) return TQ_ERR_CUDA;
    const int threads = D == 128 ? AppendRoles<128>::kThreads : AppendRoles<64>::kThreads;
    if (w == 1 && axes) p.f = HeadXform{}, p.pos = nullptr;    // values are not turned: no positions looked up
    if (const int rc = launch_one(fn, grid, threads, kSmem, st, p, w, w == 1, "tq_append_ragged"))
      return rc;
  }
  return TQ_OK;
}

int launch_dequant_ragged_tc(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                             const tq_ragged* batch, const tq_tensor4* ko, const tq_tensor4* vo,
                             uint32_t* status, cudaStream_t st) {
  const int D = G->head_dim;
  const tq_tensor4* x[2] = {ko, vo};
  const tq_tensor4* one = ko ? ko : vo;
  if (D != 64 && D != 128) return 1;
  if (one->shape[1] * one->shape[2] > INT32_MAX - kM) return 1;
  if (reinterpret_cast<uintptr_t>(t->rot) % 16) return 1;
  RaggedTc p = tc_params(G, t, c, x, batch, status);
  const unsigned grid = (unsigned)tmin(p.ntiles, device_sm_count());
  for (int w = 0; w < 2; ++w) {
    if (!x[w]) continue;
    p.vec[w] = rows_aligned(x[w]);
    const int bits = w == 0 ? G->key_bits : G->value_bits;
    int bytes = 0;
    const bool lo = x[w]->dtype != TQ_BF16;
    RaggedFn fn = D == 128 ? (lo ? read_fn<128, true>(bits, bytes) : read_fn<128, false>(bits, bytes))
                           : (lo ? read_fn<64, true>(bits, bytes) : read_fn<64, false>(bits, bytes));
    if (set_smem_attr((const void*)fn, bytes) != TQ_OK) return TQ_ERR_CUDA;
    const int threads = D == 128 ? ReadRoles<128>::kThreads : ReadRoles<64>::kThreads;
    if (const int rc = launch_one(fn, grid, threads, bytes, st, p, w, w == 1 && ko,
                                  "tq_dequantize_ragged"))
      return rc;
  }
  return TQ_OK;
}

}  // namespace tq
