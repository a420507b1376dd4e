// tq_attend_pair.cu — differential attention with keys of each map's own, off the packed
// pages, for few query rows per request and pair of KV heads (tq_diff_attend_ragged):
//   out = out_scale norm(A1 [V1 V2] - lambda A2 [V1 V2]),  Am = softmax(q_m K_m^T)
//
// A CTA holds 8 rows (positions x pairs of query heads of one pair of KV heads) of both
// maps and a range of pages of both heads; its four warps take a quarter (16 tokens) of
// every page, as in tq_attend_few.cu, whose fragments and tables these are.  Per tile of
// 16 tokens, tokens on M and the 8 rows of a map on N of mma.sync m16n8k16:
//   S_m^T = K^_m Q'_m^T                    one product a map
//   O_hm^T += V^_h^T P'_hm^T               both maps on the same decoded values
// so every code is looked up once for both maps: 4 lookups of a row's codes (two keys, two
// values), where a map at a time takes 6 and a (map, half of the values) at a time 8.  The
// result's 16 D values per row and thread group are 128 registers (D = 128), so two CTAs
// share an SM, and a page's codes are loaded into the registers of the last page's as
// soon as those are used up.
//
// The two maps' sums meet at the end of a row: u = O_1 / l_1 - lambda O_2 / l_2 in the
// rotated basis, where the norm's sum of squares is the same, then out = u R: 8 rows x 2
// halves are the 16 rows of one MMA tile.
//
// Bound by the lookups' shared-memory wavefronts and latency, as tq_attend_few.cu.  4 pairs of
// KV heads of 128, g 4, K4/V2: single tokens of 64 requests over 235,555 keys 121 us, 1.6
// TB/s (2,017 us with a (map, half) at a time on mma.sync tiles of 128 rows); one token
// over 500 keys 31 us, over 65,000 80.  K4/V4, 8,193 rows of prompt chunks 2.9 ms against
// 4.1: ahead of those tiles at any number of rows (16 a map and request 96 us against 453,
// 128 321 against 540, 2,048 4,670 against 7,174).  HP multiplies three times and reads
// eight bytes a lookup; it spills up to 52 bytes a thread, with heads of 64 up to 92.  Of the
// bf16 instances K4/V2 and K4/V4 of 128 spill 20 and 16.
#include "tq_attend_few.cuh"
#include "tq_internal.h"

#include <limits.h>
#include <math.h>
#include <type_traits>

namespace tq {
namespace {
using namespace few;

struct PairParams {
  const uint8_t* pages;
  PageMap pm;
  int nblocks;                  // pages that a table entry may name
  int page_bytes, off_v, off_kn, off_vn;
  const __half* rot_h;          // R [D][D] fp16
  const float* rot;             // R [D][D] (HP)
  const __half* qp;             // q' rows (ragged_plan_kernel), [token][Hq][D] in quad order; HP: [2][D], hi and lo
  int64_t qp_stride;            // tokens of q' per request; 0: q' follows the batch's rows
  const float* kc;
  const float* vc;
  void* out; int o_dtype; int o_pair; int64_t os[3];   // head, row, dim; pairs in one store
  int g, hc, nchunk, pcta;      // pairs of query heads per pair of KV heads, per CTA
  int Hq;
  int causal;
  const float* lambda; int64_t ls[2];
  const void* w; int w_dtype;   // the norm's weight or NULL: no norm
  float eps, offset, out_scale;
  uint32_t* status;
  RaggedAttend rg;
};

constexpr int kRows = 8;        // query rows of a CTA and map

template <int D, int KB, int VB, bool HP>
struct Pair {
  static constexpr bool KQ = KB == 2 && !HP, VQ = VB == 2 && !HP;   // two pairs per table entry
  static constexpr int KT = 128 << (KQ ? 8 : 2 * KB), VT = 128 << (VQ ? 8 : 2 * VB);   // tables
  static constexpr int W = 2 * D, LDO = W + 4;              // floats per row of an output (banks)
  static constexpr int LDA = D / 2 + 4;                     // words per row of a rotation operand
  // after the loop the tables are dead: partial outputs, then the joined one (in the
  // first's place), R and the operand of the last rotation over the others
  static constexpr int OFF_P = 0;                           // [kW][16][LDO]
  static constexpr int OFF_ROT = (16 * LDO * 4 + 127) & ~127;
  static constexpr int OFF_A = OFF_ROT + 2 * D * D;         // [hi, lo][16][LDA]
  static constexpr int LOOP = KT + VT, END = tmax(kW * 16 * LDO * 4, OFF_A + 2 * 16 * LDA * 4);
  static constexpr int OFF_Q = (tmax(LOOP, END) + 127) & ~127;      // q' fp16 [2][8][D]
  static constexpr int OFF_M = OFF_Q + (HP ? 2 : 1) * 16 * D * 2;   // (HP: and lo); [kW][16] running max
  static constexpr int OFF_L = OFF_M + kW * 16 * 4;         // [kW][16] sums
  static constexpr int OFF_R = OFF_L + kW * 16 * 4;         // [16] sums, [16] maxima, flags, limits
  static constexpr int BYTES = OFF_R + 256;
  static constexpr int kBatch = (OFF_Q - OFF_A) / (8 * 16); // parts whose {m, l} are staged at once
  static_assert(kBatch >= 16, "room for a batch of parts");
};

// A page of both heads: codes and norms of the thread's tokens.
template <int D, int KB, int VB>
struct PairTile {
  static constexpr int KN = D / 4 * KB / 8, VN = D / 8 * VB / 8;
  Codes<KN> k[2][2];            // [head]: tokens gq, gq + 8: quad tq
  Codes<VN> v[2][4];            // [head]: tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9: octet gq
  uint16_t kn[2][2], vn[2][2];  // fp16 norms of tokens gq, gq + 8
};

template <int D, int KB, int VB, bool HP>
__device__ __forceinline__ void fill_tables(const PairParams& p, unsigned char* sm) {
  using F = Pair<D, KB, VB, HP>;
  fill_table<KB, F::KQ, HP>(sm, p.kc, threadIdx.x, 32 * kW);
  fill_table<VB, F::VQ, HP>(sm + F::KT, p.vc, threadIdx.x, 32 * kW);
}

// One segment of the work list.
template <int D, int KB, int VB, bool HP>
__device__ __forceinline__ void attend_segment(const PairParams& p, const SegWork& sw,
                                               unsigned char* sm, bool filled) {
  using F = Pair<D, KB, VB, HP>;
  using Tile = PairTile<D, KB, VB>;
  constexpr int NC = D / 16, kThreads = 32 * kW, LDA = F::LDA, LDO = F::LDO, W = F::W;
  constexpr int KROW = D * KB / 8, VROW = D * VB / 8;
  float* mw = reinterpret_cast<float*>(sm + F::OFF_M);
  float* lw = reinterpret_cast<float*>(sm + F::OFF_L);
  float* U = reinterpret_cast<float*>(sm + F::OFF_P);
  uint32_t* A = reinterpret_cast<uint32_t*>(sm + F::OFF_A);
  float* rowl = reinterpret_cast<float*>(sm + F::OFF_R);
  int* flags = reinterpret_cast<int*>(sm + F::OFF_R + 128);   // last CTA, first bad key
  int* lims = reinterpret_cast<int*>(sm + F::OFF_R + 192);    // [8] last key each row sees

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  const HeadView& hv = p.rg.hv;
  const int kvp = sw.group / p.nchunk, chunk = sw.group % p.nchunk;
  const int h0 = kvp * p.g + chunk * p.hc;                 // first pair of query heads
  const int nh = min(p.hc, p.g - chunk * p.hc);            // pairs of this CTA
  const int64_t stream0 = (int64_t)sw.seg.req * hv.streams;
  const int q_len = (int)sw.rq.q_len, pos0 = sw.seg.tile * p.pcta;
  // keys in the pages, position of the request's row 0: 32 bits (base + q_len is a length)
  const int seq = (int)sw.rq.seq, t_base = (int)sw.rq.base;
  // row n of the CTA: position pos0 + n / hc, pair h0 + n % hc
  auto row_pos = [&](int n) { return n < p.pcta * p.hc ? pos0 + n / p.hc : INT_MAX; };
  auto row_valid = [&](int n) { return row_pos(n) < q_len && n % p.hc < nh; };
  // the last key row n sees
  auto row_lim = [&](int n) -> int {
    return p.causal && row_valid(n) ? min(t_base + row_pos(n), seq - 1) : seq - 1;
  };
  const int kend = p.causal ? max(min(t_base + min(pos0 + p.pcta, q_len), seq), 0) : seq;

  // ---- the thread's place in every page and the first pages' loads -------------
  uint32_t ksh, vsh;
  const int s0 = 16 * warp;                                // first token of the quarter
  const int at_k = (s0 + gq) * KROW + code_start<Tile::KN>(tq * Tile::KN, ksh);
  const int at_v = p.off_v + (s0 + 2 * tq) * VROW + code_start<Tile::VN>(gq * Tile::VN, vsh);
  const int at_n = p.off_kn + 2 * (s0 + gq);
  const int pend = min(sw.seg.kt1, (kend + 63) >> 6);      // pages [kt0, pend)
  const int64_t st[2] = {stream0 + hv.kv_pair(kvp, 0), stream0 + hv.kv_pair(kvp, 1)};
  auto entry = [&](int s, int pg) -> int {
    pg = min(pg, pend - 1);
    return p.pm.bt ? __ldg(p.pm.bt + st[s] * p.pm.bt_stride + pg) : (int)(st[s] * p.pm.pps) + pg;
  };
  auto checked = [&](int e) -> int {
    if ((unsigned)e < (unsigned)p.nblocks) return e;       // e < 0 is not
    atomicOr(p.status, TQ_DEV_BAD_BLOCK);
    return 0;
  };
  Tile x;
  auto load_keys = [&](int s, int e) {
    const uint8_t* page = page_at(p.pages, e, p.page_bytes);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.k[s][i].load(page + at_k + 8 * i * KROW);
      x.kn[s][i] = __ldg(reinterpret_cast<const uint16_t*>(page + at_n + 16 * i));
      x.vn[s][i] = __ldg(reinterpret_cast<const uint16_t*>(page + at_n + 128 + 16 * i));
    }
  };
  auto load_values = [&](int s, int e) {
    const uint8_t* v = page_at(p.pages, e, p.page_bytes) + at_v;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[s][i].load(v + ((i & 1) + 8 * (i >> 1)) * VROW);
  };
  int pg = sw.seg.kt0;
  const bool any = pg < pend;
  int e_next[2] = {0, 0}, e_after[2] = {0, 0};
  if (any) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int e = checked(entry(s, pg));
      e_next[s] = entry(s, pg + 1);
      e_after[s] = entry(s, pg + 2);
      load_keys(s, e);
      load_values(s, e);
    }
  }

  // ---- query rows, table ---------------------------------------------------------
  if (tid == 0) flags[1] = INT_MAX;
  if (tid < kRows) lims[tid] = row_lim(tid);
  // 16-byte piece k of row n (8 m + row), quad t of q' (quad order): its place in the row
  auto q_piece = [](int n, int t, int k) {
    const int f = D == 128 ? ((t >> 1) | ((n & 1) << 1)) : (n & 1);
    return n * (D / 8) + t * (D / 32) + (k ^ f);
  };
  const int64_t tok0 = p.qp_stride ? sw.seg.req * p.qp_stride : sw.rq.q0;
  constexpr int kQLo = 16 * D * 2;                         // HP: lo behind hi
#pragma unroll
  for (int part = 0; part < (HP ? 2 : 1); ++part)
    for (int i = tid; i < 16 * D / 8; i += kThreads) {
      const int n = i / (D / 8), c = i % (D / 8), row = n & 7, m = n >> 3;
      unsigned char* dst = sm + F::OFF_Q + part * kQLo + 16 * q_piece(n, c / (D / 32), c % (D / 32));
      if (row_valid(row))
        cp_async16(dst, p.qp + ((tok0 + row_pos(row)) * p.Hq + hv.in_q(2 * (h0 + row % p.hc) + m)) *
                                   (HP ? 2 * D : D) + part * D + 8 * c);
      else
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
    }
  if (!filled) fill_tables<D, KB, VB, HP>(p, sm);
  cp_async_wait_all();
  __syncthreads();

  // ---- pages -----------------------------------------------------------------------
  float O[2][NC][2][4];                                    // [half][chunk of D][map]
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) O[h][i][n][0] = O[h][i][n][1] = O[h][i][n][2] = O[h][i][n][3] = 0.f;
  float m[2][2], l[2][2];                                  // [map][column]
  float vs[2] = {4194304.f, 4194304.f};                    // scales of the value norms, 2^22 at most
  const int lim[2] = {lims[2 * tq], lims[2 * tq + 1]};
  int lim_min = min(lim[0], lim[1]);
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = kNoMax;
      l[n][c] = 0.f;
    }
  const uint32_t k_base = smem_u32(sm) + (F::KQ || HP ? 8 * (lane & 15) : 4 * lane);
  const uint32_t v_base = smem_u32(sm + F::KT) + (F::VQ || HP ? 8 * (lane & 15) : 4 * lane);
  int bad_key = INT_MAX;

#pragma unroll 1
  for (; pg < pend; ++pg) {
    const int en[2] = {checked(e_next[0]), checked(e_next[1])};
    if (lane == 0 && warp < 2 && (unsigned)e_after[warp] < (unsigned)p.nblocks)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                   ::"l"(page_at(p.pages, warp ? e_after[1] : e_after[0], p.page_bytes)),
                     "r"(p.page_bytes) : "memory");
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      e_next[s] = e_after[s];
      e_after[s] = entry(s, pg + 3);
    }
    const int key0 = 64 * pg + s0 + gq;
    // norms: 0 past the end; a token with a norm that is not finite counts as 0 (0 x inf
    // would reach rows that do not see it) and the rows that see it become NaN at the end
    float kn[2][2], vn[2][2], s[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t u = (uint32_t)x.kn[h][i] | ((uint32_t)x.vn[h][i] << 16);
        const bool in = key0 + 8 * i < kend;
        // exponent 31 in either half carries into its sign bit
        const bool fin = (((u & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u) == 0;
        if (in && !fin) bad_key = min(bad_key, key0 + 8 * i);
        u = in && fin ? u : 0u;
        const __half2 h2 = *reinterpret_cast<const __half2*>(&u);
        kn[h][i] = __low2float(h2);
        vn[h][i] = __high2float(h2) * vs[h];
      }
    // S_m^T, m by m: two chunks of 16 dims share one 16-byte piece of q'
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      uint32_t kw[2][Codes<Tile::KN>::NW];
      x.k[n][0].words(kw[0], ksh);
      x.k[n][1].words(kw[1], ksh);
      if (F::KQ) join_nibbles(kw[0], kw[1]);
#pragma unroll
      for (int c2 = 0; c2 < NC / 2; ++c2) {
        const unsigned char* at = sm + F::OFF_Q + 16 * q_piece(8 * n + gq, tq, c2);
        const uint4 qb = *reinterpret_cast<const uint4*>(at);
        uint4 ql = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (HP) ql = *reinterpret_cast<const uint4*>(at + kQLo);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t a[4], al[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = 2 * (2 * c2 + c) + i;
            if constexpr (HP)
              look_up_split<2 * KB>(k_base, kw[0], kw[1], k, a[2 * i], a[2 * i + 1], al[2 * i], al[2 * i + 1]);
            else
              look_up2<2 * KB, F::KQ>(k_base, kw[0], kw[1], k, a[2 * i], a[2 * i + 1]);
          }
          mma_f16_16816(s[n], a, c ? qb.z : qb.x, c ? qb.w : qb.y);
          if constexpr (HP) {
            mma_f16_16816(s[n], a, c ? ql.z : ql.x, c ? ql.w : ql.y);
            mma_f16_16816(s[n], al, c ? qb.z : qb.x, c ? qb.w : qb.y);
          }
        }
      }
      load_keys(n, en[n]);                                 // the next page's, into what is used up
    }
    // relative to m
    float d[2][4], top = -INFINITY;
    const bool edge = 64 * pg + s0 + 15 > lim_min;
    auto hidden = [&](int i, int c) { return key0 + 8 * i > lim[c]; };
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[n][i] = fmaf(s[n][i], kn[n][i >> 1], -m[n][i & 1]);
    if (edge) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hidden(i >> 1, i & 1)) d[n][i] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) top = fmaxf(fmaxf(fmaxf(top, d[n][0]), fmaxf(d[n][1], d[n][2])), d[n][3]);
    const float big[2] = {fmaxf(fabsf(vn[0][0]), fabsf(vn[0][1])), fmaxf(fabsf(vn[1][0]), fabsf(vn[1][1]))};
    if (__any_sync(0xffffffffu, top > kRoom || fmaxf(big[0], big[1]) >= kNorm)) {
      // each half's largest norm of the tile, below 2^(e + 1): down to below kNorm
      float r[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(big[h])) >> 23) - 127;
        r[h] = __uint_as_float((uint32_t)(127 - max(e - 7, 0)) << 23);
        vs[h] *= r[h];
        vn[h][0] *= r[h];
        vn[h][1] *= r[h];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // the largest score of the column in this tile
          const bool out0 = edge && hidden(0, c), out1 = edge && hidden(1, c);
          float y = fmaxf(out0 ? -INFINITY : s[n][c] * kn[n][0], out1 ? -INFINITY : s[n][2 + c] * kn[n][1]);
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
          const float mn = fmaxf(m[n][c], y), f = fast_exp2(m[n][c] - mn);
          l[n][c] *= f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < NC; ++i) { O[h][i][n][c] *= f * r[h]; O[h][i][n][2 + c] *= f * r[h]; }
          m[n][c] = mn;
          d[n][c] = out0 ? -INFINITY : fmaf(s[n][c], kn[n][0], -mn);
          d[n][2 + c] = out1 ? -INFINITY : fmaf(s[n][2 + c], kn[n][1], -mn);
        }
    }
    float pr[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[n][i] = fast_exp2(d[n][i]);
        l[n][i & 1] += pr[n][i];
      }
    constexpr int VW = Codes<Tile::VN>::NW;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t pb[2][2], pl[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = pr[n][2 * i] * vn[h][i], p1 = pr[n][2 * i + 1] * vn[h][i];
          if constexpr (HP) {
            uint32_t lo;
            pb[n][i] = movmatrix_trans(split2(p0, p1, lo));
            pl[n][i] = movmatrix_trans(lo);
          } else {
            pb[n][i] = movmatrix_trans(pack_half2(p0, p1));
          }
        }
      uint32_t ve[2][VW], vo[2][VW];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t a[VW], b[VW];
        x.v[h][2 * i].words(a, vsh);
        x.v[h][2 * i + 1].words(b, vsh);
        join_tokens<VB>(a, b, ve[i], vo[i]);
        if (F::VQ) join_nibbles(ve[i], vo[i]);
      }
      load_values(h, en[h]);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t a[4], al[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (HP)
            look_up_split<2 * VB>(v_base, ve[i], vo[i], c, a[2 * i], a[2 * i + 1], al[2 * i], al[2 * i + 1]);
          else
            look_up2<2 * VB, F::VQ>(v_base, ve[i], vo[i], c, a[2 * i], a[2 * i + 1]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mma_f16_16816(O[h][c][n], a, pb[n][0], pb[n][1]);
          if constexpr (HP) {
            mma_f16_16816(O[h][c][n], a, pl[n][0], pl[n][1]);
            mma_f16_16816(O[h][c][n], al, pb[n][0], pb[n][1]);
          }
        }
      }
    }
  }
  if (bad_key != INT_MAX) atomicMin(&flags[1], bad_key);

  // ---- the warps' partials: common max, sum in warp order; row 8 n + r is row r of map n ----
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float y = l[n][c];
      y += __shfl_xor_sync(0xffffffffu, y, 4);
      y += __shfl_xor_sync(0xffffffffu, y, 8);
      y += __shfl_xor_sync(0xffffffffu, y, 16);
      if (gq == 0) {
        mw[warp * 16 + 8 * n + 2 * tq + c] = m[n][c];
        lw[warp * 16 + 8 * n + 2 * tq + c] = y;
      }
    }
  __syncthreads();                                         // and the tables are dead
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * n + 2 * tq + c;
      float M = mw[row];
#pragma unroll
      for (int w = 1; w < kW; ++w) M = fmaxf(M, mw[w * 16 + row]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // times 1 / vs (exponents: vs is a power of two)
        const float f = fast_exp2(m[n][c] - M) * __uint_as_float(0x7F000000u - __float_as_uint(vs[h]));
        float* mine = U + (warp * 16 + row) * LDO + h * D + gq;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          mine[16 * i] = O[h][i][n][c] * f;
          mine[16 * i + 8] = O[h][i][n][2 + c] * f;
        }
      }
    }
  if (tid < 16) {
    float M = mw[tid], y = 0.f;
#pragma unroll
    for (int w = 1; w < kW; ++w) M = fmaxf(M, mw[w * 16 + tid]);
#pragma unroll
    for (int w = 0; w < kW; ++w) y += lw[w * 16 + tid] * fast_exp2(mw[w * 16 + tid] - M);
    if (flags[1] <= row_lim(tid & 7)) y = NAN;
    rowl[tid] = y;
    rowl[16 + tid] = M;
  }
  __syncthreads();
  for (int i = tid; i < 16 * W / 4; i += kThreads) {
    const int at = i / (W / 4) * LDO + 4 * (i % (W / 4));
    float4 a = *reinterpret_cast<const float4*>(U + at);
#pragma unroll
    for (int w = 1; w < kW; ++w) {
      const float4 b = *reinterpret_cast<const float4*>(U + w * 16 * LDO + at);
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    *reinterpret_cast<float4*>(U + at) = a;
  }
  __syncthreads();
  // R for the last rotation, on its way while a split tile's parts come together
  for (int i = tid; i < D * D / 8; i += kThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    unsigned char* dst = sm + F::OFF_ROT + r * (2 * D) + ((c ^ (r & 7)) << 4);
    if constexpr (HP) {                                    // lo first
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = __ldg(reinterpret_cast<const float2*>(p.rot + 8 * i) + e);
        split2(y.x, y.y, w[e]);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      cp_async16(dst, p.rot_h + 8 * i);
    }
  }

  // ---- a split tile: partials out, the last CTA joins them -----------------------
  if (sw.seg.slot >= 0) {
    const RaggedPlan& pl = p.rg.plan;
    for (int i = tid; i < 16 * W / 4; i += kThreads) {
      const int n = i / (W / 4), at = 4 * (i % (W / 4));
      if (row_valid(n & 7))
        *reinterpret_cast<float4*>(pl.part + part_row(pl, sw.seg.slot, sw.group, n) * W + at) =
            *reinterpret_cast<const float4*>(U + n * LDO + at);
    }
    if (tid < 16) pl.ml[part_row(pl, sw.seg.slot, sw.group, tid)] = make_float2(rowl[16 + tid], rowl[tid]);
    if (!last_of_tile(pl, sw, &flags[0])) {
      cp_async_wait_all();                                 // nothing in flight into what comes next
      return;
    }
    // batches of parts: every {m, l} in one trip, then the weights 2^(m - M); parts come in
    // slot order whatever the order of arrival
    const int parts = sw.seg.parts;
    float2* wl = reinterpret_cast<float2*>(sm + F::OFF_A);   // [parts][16] of a batch
    constexpr int NE = 16 * W / 4 / kThreads;              // float4 columns per thread
    float4 acc[NE];
#pragma unroll
    for (int k = 0; k < NE; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    float run_m = kNoMax, run_l = 0.f;                     // of row tid (tid < 16)
    for (int b0 = 0; b0 < parts; b0 += F::kBatch) {
      const int ns = min(F::kBatch, parts - b0);
      for (int i = tid; i < ns * 16; i += kThreads)
        wl[i] = __ldcg(pl.ml + part_row(pl, sw.seg.first + b0 + i / 16, sw.group, i % 16));
      __syncthreads();
      if (tid < 16) {
        float M = run_m;
        for (int s = 0; s < ns; ++s) M = fmaxf(M, wl[s * 16 + tid].x);
        const float f = fast_exp2(run_m - M);              // of what earlier batches left
        run_l *= f;
        for (int s = 0; s < ns; ++s) {
          const float w = fast_exp2(wl[s * 16 + tid].x - M);
          run_l = fmaf(w, wl[s * 16 + tid].y, run_l);
          wl[s * 16 + tid].x = w;
        }
        run_m = M;
        rowl[tid] = f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NE; ++k) {
        const int i = tid + k * kThreads, n = i / (W / 4);
        const float f = rowl[n];
        acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
        if (!row_valid(n & 7)) continue;
        const float* src = pl.part + part_row(pl, sw.seg.first + b0, sw.group, n) * W + 4 * (i % (W / 4));
#pragma unroll 4
        for (int s = 0; s < ns; ++s) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(src + s * ((int64_t)pl.G * pl.rows * W)));
          const float w = wl[s * 16 + n].x;
          acc[k].x = fmaf(w, y.x, acc[k].x);
          acc[k].y = fmaf(w, y.y, acc[k].y);
          acc[k].z = fmaf(w, y.z, acc[k].z);
          acc[k].w = fmaf(w, y.w, acc[k].w);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int i = tid + k * kThreads;
      *reinterpret_cast<float4*>(U + i / (W / 4) * LDO + 4 * (i % (W / 4))) = acc[k];
    }
    if (tid < 16) rowl[tid] = run_l;
    __syncthreads();
  }

  // ---- u = out_scale norm(O_1 / l_1 - lambda O_2 / l_2), half h of row r as row 8 h + r of the
  // rotation's operand, each times the power of two that puts its largest value into
  // [2^10, 2^11), which the result is divided by.  A warp takes two rows.
#pragma unroll
  for (int r0 = 0; r0 < kRows; r0 += kW) {
    const int r = r0 + warp;
    const bool valid = row_valid(r);
    const float l1 = valid ? rowl[r] : 0.f, l2 = valid ? rowl[8 + r] : 0.f;
    const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : 1.f / l2;
    float lambda = 0.f;
    if (valid)
      lambda = __ldg(p.lambda + (sw.rq.q0 + row_pos(r)) * p.ls[0] + (h0 + r % p.hc) * p.ls[1]);
    auto diff = [&](float a, float b) {
      a *= i1;
      b *= i2;
      return b == 0.f ? a : fmaf(-lambda, b, a);           // rows without keys are 0
    };
    float2 u[2][D / 64];
    float ss = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        u[h][k] = make_float2(0.f, 0.f);
        if (valid) {
          const int at = h * D + 2 * (lane + 32 * k);
          const float2 a = *reinterpret_cast<const float2*>(U + r * LDO + at);
          const float2 b = *reinterpret_cast<const float2*>(U + (8 + r) * LDO + at);
          u[h][k] = make_float2(diff(a.x, b.x), diff(a.y, b.y));
        }
        ss = fmaf(u[h][k].x, u[h][k].x, fmaf(u[h][k].y, u[h][k].y, ss));
      }
    float f = p.out_scale;
    if (p.w) {
      ss = warp_sum(ss);
      f = ss == 0.f ? 0.f : f / sqrtf(fmaf(ss, 1.f / (float)W, p.eps));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        u[h][k].x *= f;
        u[h][k].y *= f;
        top = fmaxf(top, fmaxf(fabsf(u[h][k].x), fabsf(u[h][k].y)));
      }
      // (a row of NaN has none: the maximum leaves NaN out; of zeros neither)
      const int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
      const int up = e == 128 ? 0 : min(10 - e, 100);
      const float sc = __uint_as_float((uint32_t)(127 + up) << 23);
      const int n = 8 * h + r;
      if (lane == 0) rowl[16 + n] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const int w = lane + 32 * k;
        A[n * LDA + w] = split2(u[h][k].x * sc, u[h][k].y * sc, A[(16 + n) * LDA + w]);
      }
    }
  }
  cp_async_wait_all();
  __syncthreads();
  // ---- out = u R -------------------------------------------------------------------
  const bool o_ok = row_valid(gq);
  const int64_t o_at = o_ok ? (sw.rq.q0 + row_pos(gq)) * p.os[1] + (int64_t)(h0 + gq % p.hc) * p.os[0] : 0;
  const float o_inv[2] = {rowl[16 + gq], rowl[24 + gq]};
  constexpr int NJ = D / 8 / kW;
  // HP: O^hi R^lo first, then the place's other half
  float lo[HP ? NJ : 1][4];
  if constexpr (HP) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      lo[j][0] = lo[j][1] = lo[j][2] = lo[j][3] = 0.f;
      rotate_slice<D, false>(lo[j], sm + F::OFF_ROT, A, warp + kW * j, lane);
    }
    __syncthreads();
    for (int i = tid; i < D * D / 8; i += kThreads) {
      const int r = i / (D / 8), c = i % (D / 8);
      cp_async16(sm + F::OFF_ROT + r * (2 * D) + ((c ^ (r & 7)) << 4), p.rot_h + 8 * i);
    }
    cp_async_wait_all();
    __syncthreads();
  }
#pragma unroll(HP ? NJ : 1)
  for (int j = 0; j < NJ; ++j) {
    const int jt = warp + kW * j;
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (HP)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = lo[j][i];
    rotate_slice<D, true>(c, sm + F::OFF_ROT, A, jt, lane);
    if (!o_ok) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = h * D + 8 * jt + 2 * tq;
      float y = c[2 * h] * o_inv[h], z = c[2 * h + 1] * o_inv[h];
      if (p.w) {
        y *= load_elem(p.w, p.w_dtype, col) + p.offset;
        z *= load_elem(p.w, p.w_dtype, col + 1) + p.offset;
      }
      const int64_t o = o_at + (int64_t)col * p.os[2];
      if (p.o_pair) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(y, z);
        reinterpret_cast<uint32_t*>(p.out)[o >> 1] =
            p.o_dtype == TQ_BF16 ? *reinterpret_cast<const uint32_t*>(&b) : pack_half2(y, z);
      } else {
        store_elem(p.out, p.o_dtype, o, y);
        store_elem(p.out, p.o_dtype, o + p.os[2], z);
      }
    }
  }
}

template <int D, int KB, int VB, bool HP>
__global__ void __launch_bounds__(32 * kW, D == 128 ? 2 : 3) attend_pair_kernel(PairParams p) {
  extern __shared__ __align__(128) unsigned char sm[];
  // segments in the list's order (long ones first), whoever is free next
  __shared__ int next;
  bool filled = true;
  fill_tables<D, KB, VB, HP>(p, sm);                       // beside the launch before
  pdl_wait();                                              // the list and q'
  for (;; filled = false) {
    __syncthreads();                                       // the last segment is done with
    if (threadIdx.x == 0) next = atomicAdd(p.rg.plan.next, 1);
    __syncthreads();
    SegWork sw;
    if (!take_segment(p.rg, next, sw)) return;
    attend_segment<D, KB, VB, HP>(p, sw, sm, filled);
  }
}
using PairFn = void (*)(PairParams);

template <int D, bool HP>
PairFn pair_fn(int kb, int vb, int& bytes) {
#define TQ_PAIR(K, V) \
  if (kb == K && vb == V) { bytes = Pair<D, K, V, HP>::BYTES; return attend_pair_kernel<D, K, V, HP>; }
  TQ_PAIR(4, 2) TQ_PAIR(4, 3) TQ_PAIR(4, 4) TQ_PAIR(3, 2) TQ_PAIR(3, 3) TQ_PAIR(3, 4)
  TQ_PAIR(2, 2) TQ_PAIR(2, 3) TQ_PAIR(2, 4)
#undef TQ_PAIR
  return nullptr;
}

}  // namespace

bool attend_pair_applies(const tq_geom* G) {
  int bytes;
  if (G->head_dim == 128) return pair_fn<128, false>(G->key_bits, G->value_bits, bytes) != nullptr;
  if (G->head_dim == 64) return pair_fn<64, false>(G->key_bits, G->value_bits, bytes) != nullptr;
  return false;
}

int launch_attend_pair(const tq_geom* G, const tq_tables* t, const tq_cache* c, const tq_diff_args* a,
                       bool precise, const RaggedAttend& rg, int hc, int pcta, const __half* qp,
                       int64_t qp_stride, int64_t grid, uint32_t* status, cudaStream_t st) {
  PairParams p = {};
  const PageGeom g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.pages = c->pages;
  p.pm = page_map(c);
  p.nblocks = p.pm.bt ? (int)p.pm.nblocks : INT_MAX;
  p.page_bytes = g.page_bytes;
  p.off_v = g.off_v;
  p.off_kn = g.off_kn;
  p.off_vn = g.off_vn;
  p.rot_h = reinterpret_cast<const __half*>(t->rot_f16);
  p.rot = t->rot;
  p.qp = qp;
  p.qp_stride = qp_stride;
  p.kc = t->k_centroids;
  p.vc = t->v_centroids;
  p.Hq = (int)a->q->shape[1];
  p.out = a->out->data; p.o_dtype = a->out->dtype;
  for (int i = 0; i < 3; ++i) p.os[i] = a->out->stride[i + 1];
  p.o_pair = p.o_dtype != TQ_F32 && p.os[2] == 1 && reinterpret_cast<uintptr_t>(p.out) % 4 == 0 &&
             (a->out->shape[1] == 1 || p.os[0] % 2 == 0) && (a->out->shape[2] == 1 || p.os[1] % 2 == 0);
  p.g = rg.hv.g;
  p.hc = hc;
  p.nchunk = (p.g + hc - 1) / hc;
  p.pcta = pcta;
  p.causal = a->causal;
  p.lambda = a->lambda;
  for (int i = 0; i < 2; ++i) p.ls[i] = a->lambda_stride[i];
  if (a->norm) {
    p.w = a->norm->weight;
    p.w_dtype = a->norm->dtype;
    p.eps = a->norm->eps;
    p.offset = a->norm->offset;
  }
  p.out_scale = a->out_scale;
  p.status = status;
  p.rg = rg;
  int bytes = 0;
  const int kb = G->key_bits, vb = G->value_bits;
  const PairFn fn = G->head_dim == 128 ? (precise ? pair_fn<128, true>(kb, vb, bytes) : pair_fn<128, false>(kb, vb, bytes))
                                       : (precise ? pair_fn<64, true>(kb, vb, bytes) : pair_fn<64, false>(kb, vb, bytes));
  if (set_smem_attr((const void*)fn, bytes) != TQ_OK) return TQ_ERR_CUDA;
  // CTAs that fit at once
  const int64_t fit = (int64_t)device_sm_count() * occupancy((const void*)fn, 32 * kW, bytes);
  return launch_result(launch_pdl(fn, dim3((unsigned)tmin(grid, fit)), dim3(32 * kW), bytes, st, p),
                       "tq_diff_attend_ragged/pair");
}

}  // namespace tq
