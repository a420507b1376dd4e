// tq_attend_few.cu — ragged attention off the packed pages for few query rows
// per request and KV head: single tokens, draft verification, short chunks.
//
// A CTA holds NQ = 8 NT query rows (positions x heads of one GQA group) and a
// range of keys.  Its W warps take 16-token tiles in turn, each with its own
// running max, sum and output, and never meet before the end, so no barrier
// or copy pipeline stands between a warp and its loads.  Per tile:
//   S^T = K^ Q'^T  tokens on M, query rows on N: mma.sync m16n8k16 (a handful
//                  of rows would leave a 128-row tcgen05 tile empty);
//   O^T += V^^T P'^T  with P' = exp2(S n_k - m) n_v as fp16.
// A thread's codes are contiguous in a page row (quad order for K, octet order
// for V), so both operands go from one coalesced global load per row straight
// into fragment registers, through a table of code pairs: entry e is the
// half2 of pair e, copied for all 32 lanes (no bank conflicts), K pairs in the
// first and V pairs in the second 128 bytes of a 256-byte row.  The table sits
// at a multiple of 64 KB, so one byte permute (or shift + mask) of the codes
// is the whole shared-memory address.  V pairs join the codes of two tokens,
// interleaved by two masks per word.
// The running max moves only when a score passes it by kRoom (a vote; the
// shuffles and the rescale of 32 NT outputs run then: nearly every tile has a
// new max among its 16 rows, so moving it at once cost a fifth of the time).
//
// q' = scale log2(e) q R^T and out = O R run on the same MMAs with both sides
// split into fp16 hi + lo (three products, 2^-22), once per CTA and once per
// output row.
#include "tq_internal.h"
#include "tq_ragged.cuh"

#include <limits.h>
#include <math.h>
#include <type_traits>

namespace tq {
namespace {

constexpr float kLog2eF = 1.4426950408889634f;
// A score may pass the running max by this much before the max moves: p <=
// 2^7, and with a value norm of at most 2^8 P' <= 2^15 stays in fp16 (for
// larger norms the max moves at once, p <= 1 and P' <= the norm itself).
constexpr float kRoom = 7.f;

struct FewParams {
  const uint8_t* pages;
  PageMap pm;
  int page_bytes, off_v, off_kn, off_vn;
  const float* rot;             // R [D][D]
  const float* rot_t;           // R^T [D][D]
  const float* kc;
  const float* vc;
  const void* q; int q_dtype; int64_t qs[3];     // head, row, dim
  void* out; int o_dtype; int64_t os[3];
  int Hkv, g, hc, nchunk, pcta;
  float qscale;                 // softmax scale x log2(e)
  int causal;
  uint32_t* status;
  RaggedAttend rg;
};

template <int D, int NT>
struct Few {
  static constexpr int W = NT == 1 ? 16 : 12;              // warps
  static constexpr int NQ = 8 * NT;
  static constexpr int LDO = D + 4;                        // floats per row of a partial (banks)
  static constexpr int kBufs = W >= 8 ? 8 : W;             // partials summed at a time
  // offsets from a 64 KB boundary: the pair table, then (the table is dead
  // after the loop) the partial outputs over it
  static constexpr int OFF_Q = 65536;                      // q' fp16 [NQ][D]
  static constexpr int OFF_M = OFF_Q + 16 * D * 2;         // [W][NQ] running max
  static constexpr int OFF_L = OFF_M + W * NQ * 4;         // [W][NQ] sums
  static constexpr int OFF_U = OFF_L + W * NQ * 4;         // [16][LDO] joined output
  static constexpr int LDA = D / 2 + 4;                    // words per row of a rotation operand
  static constexpr int OFF_A = OFF_U + 16 * LDO * 4;       // [2: hi, lo][16][LDA] fp16 pairs
  static constexpr int OFF_R = OFF_A + 2 * 16 * LDA * 4;   // [16] sums of the rows, flags
  static constexpr int BYTES = OFF_R + 256;
  static_assert(kBufs * NQ * LDO * 4 <= 65536 + 4096, "partials");
};

// N consecutive bytes of codes as little-endian words.  Multiples of 4 are
// aligned vector loads; other counts load the words that hold them and shift.
template <int N>
struct Codes { uint32_t w[(N + 3) / 4]; };

template <int N>
__device__ __forceinline__ Codes<N> load_codes(const uint8_t* row, int off) {
  Codes<N> c;
  if constexpr (N == 16) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + off));
    c.w[0] = v.x; c.w[1] = v.y; c.w[2] = v.z; c.w[3] = v.w;
  } else if constexpr (N == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + off));
    c.w[0] = v.x; c.w[1] = v.y;
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) c.w[i] = __ldg(reinterpret_cast<const uint32_t*>(row + off) + i);
  } else if constexpr (N == 2) {
    c.w[0] = __ldg(reinterpret_cast<const uint16_t*>(row + off));
  } else {
    // 3 or 6 bytes at a multiple of 3: two words (the second may lie past the
    // row, but within the page: norms follow the codes)
    const uint32_t* p = reinterpret_cast<const uint32_t*>(row + (off & ~3));
    const uint32_t a = __ldg(p), b = __ldg(p + 1), sh = (uint32_t)(off & 3) * 8;
    c.w[0] = __funnelshift_r(a, b, sh);
    if constexpr (N > 4) c.w[1] = b >> sh;
  }
  return c;
}

// Shared address of the table row of field `k` (FB bits each, low first) of
// the words: (field << 8) | lane address.
template <int FB, int NW>
__device__ __forceinline__ uint32_t field_addr(const uint32_t (&w)[NW], int k, uint32_t lane_addr) {
  const int bo = FB * k, wi = bo >> 5, sh = bo & 31;
  if constexpr (FB == 8) {
    return __byte_perm(w[wi], lane_addr, 0x7604u | (uint32_t)((sh >> 3) << 4));
  } else {
    constexpr uint32_t mask = ((1u << FB) - 1u) << 8;
    uint32_t x;
    if (sh + FB > 32) x = __funnelshift_r(w[wi], w[wi + 1 < NW ? wi + 1 : wi], sh) << 8;
    else if (sh >= 8) x = w[wi] >> (sh - 8);
    else x = w[wi] << (8 - sh);
    return (x & mask) | lane_addr;
  }
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  return *reinterpret_cast<const uint32_t*>(__cvta_shared_to_generic(addr));
}

// Fields of two tokens' VB-bit codes joined into pairs: even entries in e, odd
// ones in o (2 VB bits each, entry 2 k (+ 1) at field k).
template <int VB, int N>
__device__ __forceinline__ void join_tokens(const Codes<N>& a, const Codes<N>& b,
                                            uint32_t (&e)[(N + 3) / 4], uint32_t (&o)[(N + 3) / 4]) {
  constexpr int NW = (N + 3) / 4;
  // VB bits of every 2 VB, continued across the words
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < 32; ++t)
      if ((((32 * i + t) / VB) & 1) == 0) m |= 1u << t;
    const uint32_t am = a.w[i] & m;
    uint32_t bl = b.w[i] << VB;                            // b's even codes up by VB
    if (i > 0) bl = __funnelshift_l(b.w[i - 1], b.w[i], VB);
    e[i] = am | (bl & ~m);
    uint32_t ar = a.w[i] >> VB;                            // a's odd codes down by VB
    if (i + 1 < NW) ar = __funnelshift_r(a.w[i], a.w[i + 1], VB);
    o[i] = (ar & m) | (b.w[i] & ~m);
  }
}

template <int D, int KB, int VB>
struct FewTile {
  static constexpr int KN = D / 4 * KB / 8, VN = D / 8 * VB / 8;
  Codes<KN> k[2];               // tokens gq, gq + 8: quad tq
  Codes<VN> v[4];               // tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9: octet gq
  uint32_t n[2];                // fp16 norms of tokens gq, gq + 8: k low, v high
};

// fp16 hi + lo of a pair (2^-22 of each value)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_half2(a, b);
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  lo = pack_half2(a - __low2float(h), b - __high2float(h));
}

// c[16 rows][8 cols] = a[16][D] M[cols][D]^T: the rows of a as fp16 pairs hi and
// lo in shared memory, M fp32 row-major with this n-tile's rows at `m`.
template <int D, int LDA>
__device__ __forceinline__ void rotate_tile(float (&c)[4], const float* m, const uint32_t* a,
                                            int lane) {
  const int gq = lane >> 2, tq = lane & 3;
  c[0] = c[1] = c[2] = c[3] = 0.f;
  float2 mv[D / 16][2];
#pragma unroll
  for (int ch = 0; ch < D / 16; ++ch) {
    mv[ch][0] = __ldg(reinterpret_cast<const float2*>(m + gq * D + 16 * ch + 2 * tq));
    mv[ch][1] = __ldg(reinterpret_cast<const float2*>(m + gq * D + 16 * ch + 2 * tq + 8));
  }
#pragma unroll
  for (int ch = 0; ch < D / 16; ++ch) {
    uint32_t bh[2], bl[2], ah[4], al[4];
    split2(mv[ch][0].x, mv[ch][0].y, bh[0], bl[0]);
    split2(mv[ch][1].x, mv[ch][1].y, bh[1], bl[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (gq + 8 * (i & 1)) * LDA + 8 * ch + tq + 4 * (i >> 1);
      ah[i] = a[at];
      al[i] = a[16 * LDA + at];
    }
    mma_f16_16816(c, ah, bh[0], bh[1]);
    mma_f16_16816(c, al, bh[0], bh[1]);
    mma_f16_16816(c, ah, bl[0], bl[1]);
  }
}

template <int D, int KB, int VB, int NT>
__global__ void __launch_bounds__(32 * Few<D, NT>::W, 1) attend_few_kernel(FewParams p) {
  using F = Few<D, NT>;
  using Tile = FewTile<D, KB, VB>;
  constexpr int W = F::W, NQ = F::NQ, NC = D / 16, kThreads = 32 * W;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  SegWork sw;
  if (!take_segment(p.rg, sw)) return;
  // the table at a multiple of 64 KB of shared address space
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 65535u) & ~65535u) - raw);
  const uint32_t sbase = smem_u32(sm);
  float* mw = reinterpret_cast<float*>(sm + F::OFF_M);
  float* lw = reinterpret_cast<float*>(sm + F::OFF_L);
  float* U = reinterpret_cast<float*>(sm + F::OFF_U);
  float* rowl = reinterpret_cast<float*>(sm + F::OFF_R);
  int* flags = reinterpret_cast<int*>(sm + F::OFF_R + 128);   // last CTA, first bad key

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  const int kvh = sw.group / p.nchunk, chunk = sw.group % p.nchunk;
  const int h0 = kvh * p.g + chunk * p.hc;                 // first query head
  const int nh = min(p.hc, p.g - chunk * p.hc);            // heads of this CTA
  const int64_t stream = (int64_t)sw.seg.req * p.Hkv + kvh;
  const int q_len = (int)sw.rq.q_len, pos0 = sw.seg.tile * p.pcta;
  const int64_t seq = sw.rq.seq, t_base = seq - q_len;     // position of the request's row 0
  // row n of the CTA: position pos0 + n / hc, head h0 + n % hc
  auto row_pos = [&](int n) { return n < p.pcta * p.hc ? pos0 + n / p.hc : INT_MAX; };
  auto row_valid = [&](int n) { return row_pos(n) < q_len && n % p.hc < nh; };
  auto row_at = [&](int n, const int64_t (&s)[3]) {
    return (sw.rq.q0 + row_pos(n)) * s[1] + (int64_t)(h0 + n % p.hc) * s[0];
  };
  // the last key row n sees
  auto row_lim = [&](int n) -> int {
    return p.causal && row_valid(n) ? (int)(t_base + row_pos(n)) : (int)seq - 1;
  };
  const int kend = p.causal ? (int)max(t_base + min(pos0 + p.pcta, q_len), (int64_t)0) : (int)seq;

  // ---- table, query rows -------------------------------------------------------
  if (tid == 0) flags[1] = INT_MAX;
  for (int i = tid; i < (1 << (2 * KB)) * 8; i += kThreads) {
    const int e = i >> 3;
    const uint32_t v = pack_half2(__ldg(p.kc + (e & ((1 << KB) - 1))), __ldg(p.kc + (e >> KB)));
    reinterpret_cast<uint4*>(sm + e * 256)[i & 7] = make_uint4(v, v, v, v);
  }
  for (int i = tid; i < (1 << (2 * VB)) * 8; i += kThreads) {
    const int e = i >> 3;
    const uint32_t v = pack_half2(__ldg(p.vc + (e & ((1 << VB) - 1))), __ldg(p.vc + (e >> VB)));
    reinterpret_cast<uint4*>(sm + e * 256 + 128)[i & 7] = make_uint4(v, v, v, v);
  }
  // 16-byte piece k of row n, quad t of q' (quad order): its place in the row
  auto q_piece = [](int n, int t, int k) {
    const int f = D == 128 ? ((t >> 1) | ((n & 1) << 1)) : (n & 1);
    return n * (D / 8) + t * (D / 32) + (k ^ f);
  };
  uint32_t* A = reinterpret_cast<uint32_t*>(sm + F::OFF_A);
  constexpr int LDA = F::LDA;
  for (int i = tid; i < 16 * D / 2; i += kThreads) {
    const int n = i / (D / 2), w = i % (D / 2);
    float x = 0.f, y = 0.f;
    if (n < NQ && row_valid(n)) {
      const int64_t o = row_at(n, p.qs) + (int64_t)(2 * w) * p.qs[2];
      x = p.qscale * load_elem(p.q, p.q_dtype, o);
      y = p.qscale * load_elem(p.q, p.q_dtype, o + p.qs[2]);
    }
    split2(x, y, A[n * LDA + w], A[(16 + n) * LDA + w]);
  }
  __syncthreads();
  for (int jt = warp; jt < D / 8; jt += W) {
    float c[4];
    rotate_tile<D, LDA>(c, p.rot + 8 * jt * D, A, lane);
    // pair (8 jt + 2 tq, + 1): word jt of quad tq
    uint32_t* qw = reinterpret_cast<uint32_t*>(sm + F::OFF_Q);
    qw[4 * q_piece(gq, tq, jt >> 2) + (jt & 3)] = pack_half2(c[0], c[1]);
    if (NQ > 8) qw[4 * q_piece(gq + 8, tq, jt >> 2) + (jt & 3)] = pack_half2(c[2], c[3]);
  }
  __syncthreads();

  // ---- key tiles -------------------------------------------------------------------
  float O[NC][NT][4];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) O[i][n][0] = O[i][n][1] = O[i][n][2] = O[i][n][3] = 0.f;
  float m[NT][2], bias[NT][2], l[NT][2];
  int lim[NT][2], lim_min = INT_MAX;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = -INFINITY;
      bias[n][c] = l[n][c] = 0.f;
      lim[n][c] = row_lim(8 * n + 2 * tq + c);
      lim_min = min(lim_min, lim[n][c]);
    }
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));

  const uint32_t lane_addr = sbase + 4 * lane;
  const int tend = min(4 * sw.seg.kt1, (kend + 15) >> 4);
  auto entry = [&](int t) -> int64_t { return t < tend ? page_entry(p.pm, stream, t >> 2) : 0; };
  auto load_tile = [&](Tile& x, int64_t e, int t) {
    if (!entry_ok(p.pm, e)) {
      atomicOr(p.status, TQ_DEV_BAD_BLOCK);
      e = 0;
    }
    const uint8_t* pg = p.pages + e * (int64_t)p.page_bytes;
    const int s0 = 16 * (t & 3);                           // first token of the tile in its page
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tok = s0 + gq + 8 * i;
      x.k[i] = load_codes<Tile::KN>(pg + tok * (D * KB / 8), tq * Tile::KN);
      x.n[i] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(pg + p.off_kn) + tok) |
               ((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(pg + p.off_vn) + tok) << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = s0 + 2 * tq + (i & 1) + 8 * (i >> 1);
      x.v[i] = load_codes<Tile::VN>(pg + p.off_v + tok * (D * VB / 8), gq * Tile::VN);
    }
  };

  int t = 4 * sw.seg.kt0 + warp;
  Tile cur, nxt;
  if (t < tend) load_tile(cur, entry(t), t);
  int64_t e_next = entry(t + W);
  for (; t < tend; t += W) {
    if (t + W < tend) load_tile(nxt, e_next, t + W);
    e_next = entry(t + 2 * W);
    const int key0 = 16 * t + gq;
    float kn[2], vn[2], s[NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2 h = *reinterpret_cast<const __half2*>(&cur.n[i]);
      const bool in = key0 + 8 * i < kend;
      kn[i] = in ? __low2float(h) : 0.f;
      vn[i] = in ? __high2float(h) : 0.f;
      // 0 x inf would reach rows that do not see the key: a token whose norm is
      // not finite counts as 0 and the rows that see it become NaN at the end
      if (!(fabsf(kn[i]) + fabsf(vn[i]) < INFINITY)) {
        kn[i] = vn[i] = 0.f;
        atomicMin(&flags[1], key0 + 8 * i);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    // S^T: two chunks of 16 dims share one 16-byte piece of q'
#pragma unroll
    for (int c2 = 0; c2 < NC / 2; ++c2) {
      uint4 qb[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
        qb[n] = *reinterpret_cast<const uint4*>(sm + F::OFF_Q + 16 * q_piece(8 * n + gq, tq, c2));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a[i] = lds32(field_addr<2 * KB>(cur.k[i & 1].w, 2 * (2 * c2 + c) + (i >> 1), lane_addr));
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma_f16_16816(s[n], a, c ? qb[n].z : qb[n].x, c ? qb[n].w : qb[n].y);
      }
    }
    bool up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] *= kn[i >> 1];
    if (16 * t + 15 > lim_min) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + 8 * (i >> 1) > lim[n][i & 1]) s[n][i] = -INFINITY;
    }
    const float room[2] = {vn[0] > 256.f ? 0.f : kRoom, vn[1] > 256.f ? 0.f : kRoom};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) up = up || s[n][i] > m[n][i & 1] + room[i >> 1];
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(s[n][c], s[n][2 + c]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float mn = fmaxf(m[n][c], x);
          const float b = mn == -INFINITY ? 0.f : mn;
          const float f = fast_exp2(m[n][c] - b);          // 0 before the first key
          l[n][c] *= f;
#pragma unroll
          for (int i = 0; i < NC; ++i) { O[i][n][c] *= f; O[i][n][2 + c] *= f; }
          m[n][c] = mn;
          bias[n][c] = b;
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = fast_exp2(s[n][2 * i] - bias[n][0]);
        const float p1 = fast_exp2(s[n][2 * i + 1] - bias[n][1]);
        l[n][0] += p0;
        l[n][1] += p1;
        pb[n][i] = movmatrix_trans(pack_half2(p0 * vn[i], p1 * vn[i]));
      }
    }
    uint32_t ve[2][(Tile::VN + 3) / 4], vo[2][(Tile::VN + 3) / 4];
#pragma unroll
    for (int i = 0; i < 2; ++i) join_tokens<VB>(cur.v[2 * i], cur.v[2 * i + 1], ve[i], vo[i]);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t a[4];
      a[0] = lds32(field_addr<2 * VB>(ve[0], c, lane_addr) + 128);
      a[1] = lds32(field_addr<2 * VB>(vo[0], c, lane_addr) + 128);
      a[2] = lds32(field_addr<2 * VB>(ve[1], c, lane_addr) + 128);
      a[3] = lds32(field_addr<2 * VB>(vo[1], c, lane_addr) + 128);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16_16816(O[c][n], a, pb[n][0], pb[n][1]);
    }
    cur = nxt;
  }

  // ---- the warps' partials: common max, sum in warp order ---------------------------
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = l[n][c];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (gq == 0) {
        mw[warp * NQ + 8 * n + 2 * tq + c] = m[n][c];
        lw[warp * NQ + 8 * n + 2 * tq + c] = x;
      }
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float M = -INFINITY;
      for (int w = 0; w < W; ++w) M = fmaxf(M, mw[w * NQ + 8 * n + 2 * tq + c]);
      const float f = M == -INFINITY ? 0.f : fast_exp2(m[n][c] - M);
#pragma unroll
      for (int i = 0; i < NC; ++i) { O[i][n][c] *= f; O[i][n][2 + c] *= f; }
    }
  float* buf = reinterpret_cast<float*>(sm);
  constexpr int B = F::kBufs, LDO = F::LDO;
  auto at = [&](int n, int i, int c) {                     // O[i][n][c] of this thread
    return (8 * n + 2 * tq + (c & 1)) * LDO + 16 * i + gq + 8 * (c >> 1);
  };
#pragma unroll
  for (int round = (W - 1) / B; round >= 0; --round) {
    if (warp / B == round) {
      float* mine = buf + (warp % B) * NQ * LDO;
      const bool add = round * B + B + warp % B < W;       // a later round left its sum here
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x = O[i][n][c];
            if (add) x += mine[at(n, i, c)];
            mine[at(n, i, c)] = x;
          }
    }
    __syncthreads();
  }
  for (int i = tid; i < NQ * D; i += kThreads) {
    const int n = i / D, d = i % D;
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < B; ++w) x += buf[(w * NQ + n) * LDO + d];
    U[n * LDO + d] = x;
  }
  if (tid < NQ) {
    float M = -INFINITY, x = 0.f;
    for (int w = 0; w < W; ++w) M = fmaxf(M, mw[w * NQ + tid]);
    for (int w = 0; w < W; ++w)
      x += M == -INFINITY ? 0.f : lw[w * NQ + tid] * fast_exp2(mw[w * NQ + tid] - M);
    const int lm = row_lim(tid);
    if (flags[1] <= lm) x = NAN;
    rowl[tid] = x;
    rowl[16 + tid] = M;
  }
  __syncthreads();

  // ---- a split tile: partials out, the last CTA joins them -----------------------
  if (sw.seg.slot >= 0) {
    const RaggedPlan& pl = p.rg.plan;
    for (int i = tid; i < NQ * D / 4; i += kThreads) {
      const int n = i / (D / 4), d = 4 * (i % (D / 4));
      if (row_valid(n))
        *reinterpret_cast<float4*>(pl.part + part_row(pl, sw.seg.slot, sw.group, n) * D + d) =
            *reinterpret_cast<const float4*>(U + n * LDO + d);
    }
    if (tid < NQ) pl.ml[part_row(pl, sw.seg.slot, sw.group, tid)] = make_float2(rowl[16 + tid], rowl[tid]);
    if (!last_of_tile(pl, sw, &flags[0])) return;
    // row n's parts over the lanes of a warp for {m, l}, then its dims over them
    for (int n = warp; n < NQ; n += W) {
      if (!row_valid(n)) continue;
      float M = -INFINITY;
      for (int s = lane; s < sw.seg.parts; s += 32) {
        const float2 ml = __ldcg(pl.ml + part_row(pl, sw.seg.first + s, sw.group, n));
        M = fmaxf(M, ml.x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      float sum = 0.f, acc[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
#pragma unroll 4
      for (int s = 0; s < sw.seg.parts; ++s) {
        const int64_t pr = part_row(pl, sw.seg.first + s, sw.group, n);
        const float2 ml = __ldcg(pl.ml + pr);
        const float w = M == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        sum = fmaf(w, ml.y, sum);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(w, __ldcg(pl.part + pr * D + 32 * i + lane), acc[i]);
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) U[n * LDO + 32 * i + lane] = acc[i];
      if (lane == 0) rowl[n] = sum;
    }
    __syncthreads();
  }

  // ---- out = (O / l) R ---------------------------------------------------------------
  for (int i = tid; i < 16 * D / 2; i += kThreads) {
    const int n = i / (D / 2), w = i % (D / 2);
    float2 u = make_float2(0.f, 0.f);
    if (n < NQ && row_valid(n)) {
      const float x = rowl[n], il = x == 0.f ? 0.f : 1.f / x;
      u = *reinterpret_cast<const float2*>(U + n * LDO + 2 * w);
      u.x *= il;
      u.y *= il;
    }
    split2(u.x, u.y, A[n * LDA + w], A[(16 + n) * LDA + w]);
  }
  __syncthreads();
  int64_t o_at[2];
  bool o_ok[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int n = gq + 8 * r;
    o_ok[r] = n < NQ && row_valid(n);
    o_at[r] = o_ok[r] ? row_at(n, p.os) : 0;
  }
  for (int jt = warp; jt < D / 8; jt += W) {
    float c[4];
    rotate_tile<D, LDA>(c, p.rot_t + 8 * jt * D, A, lane);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (!o_ok[r]) continue;
      const int64_t o = o_at[r] + (int64_t)(8 * jt + 2 * tq) * p.os[2];
      store_elem(p.out, p.o_dtype, o, c[2 * r]);
      store_elem(p.out, p.o_dtype, o + p.os[2], c[2 * r + 1]);
    }
  }
}

using FewFn = void (*)(FewParams);

template <int D, int NT>
FewFn few_fn(int kb, int vb) {
#define TQ_FEW(K, V) if (kb == K && vb == V) return attend_few_kernel<D, K, V, NT>;
  TQ_FEW(4, 2) TQ_FEW(4, 3) TQ_FEW(4, 4) TQ_FEW(3, 2) TQ_FEW(3, 3) TQ_FEW(3, 4)
  TQ_FEW(2, 2) TQ_FEW(2, 3) TQ_FEW(2, 4)
#undef TQ_FEW
  return nullptr;
}

}  // namespace

bool attend_few_applies(const tq_geom* G) {
  if (G->head_dim == 128) return few_fn<128, 1>(G->key_bits, G->value_bits) != nullptr;
  if (G->head_dim == 64) return few_fn<64, 1>(G->key_bits, G->value_bits) != nullptr;
  return false;
}

int launch_attend_few(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                      const tq_attend_args* a, const RaggedAttend& rg, int64_t Hkv, int hc,
                      int pcta, int rows, int64_t grid, uint32_t* status, cudaStream_t st) {
  FewParams p;
  const PageGeom g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.pages = c->pages;
  p.pm = page_map(c);
  p.page_bytes = g.page_bytes;
  p.off_v = g.off_v;
  p.off_kn = g.off_kn;
  p.off_vn = g.off_vn;
  p.rot = t->rot;
  p.rot_t = t->rot_t;
  p.kc = t->k_centroids;
  p.vc = t->v_centroids;
  p.q = a->q->data; p.q_dtype = a->q->dtype;
  p.out = a->out->data; p.o_dtype = a->out->dtype;
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q->stride[i + 1]; p.os[i] = a->out->stride[i + 1]; }
  p.Hkv = (int)Hkv;
  p.g = (int)(a->q->shape[1] / Hkv);
  p.hc = hc;
  p.nchunk = (p.g + hc - 1) / hc;
  p.pcta = pcta;
  p.qscale = a->scale * kLog2eF;
  p.causal = a->causal;
  p.status = status;
  p.rg = rg;
  FewFn fn;
  int bytes, threads;
  auto pick = [&](auto d, auto nt) {
    constexpr int D = decltype(d)::value, NT = decltype(nt)::value;
    fn = few_fn<D, NT>(G->key_bits, G->value_bits);
    bytes = Few<D, NT>::BYTES;
    threads = 32 * Few<D, NT>::W;
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  if (G->head_dim == 128) {
    if (rows == 8) pick(std::integral_constant<int, 128>(), I1()); else pick(std::integral_constant<int, 128>(), I2());
  } else {
    if (rows == 8) pick(std::integral_constant<int, 64>(), I1()); else pick(std::integral_constant<int, 64>(), I2());
  }
  bytes += 65536;                         // slack to reach a 64 KB boundary
  if (set_smem_attr((const void*)fn, bytes) != TQ_OK) return TQ_ERR_CUDA;
  fn<<<(unsigned)grid, threads, bytes, st>>>(p);
  return check_launch("tq_attend_ragged/few");
}

}  // namespace tq
