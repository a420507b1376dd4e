// tq_attend_few.cu — ragged attention off the packed pages for few query rows
// per request and KV head: single tokens, draft verification, short chunks.
//
// A CTA holds NQ = 8 NT query rows (positions x heads of one GQA group) and a
// range of pages.  Its four warps take a quarter (16 tokens) of every page,
// each with its own running max, sum and output, and never meet before the
// end, so no barrier or copy pipeline stands between a warp and its loads;
// three CTAs share an SM, so one's set-up and end hide behind the others'
// pages.  Per tile of 16 tokens:
//   S^T = K^ Q'^T  tokens on M, query rows on N: mma.sync m16n8k16 (a handful
//                  of rows would leave a 128-row tcgen05 tile empty);
//   O^T += V^^T P'^T  with P' = exp2(S n_k - m) n_v as fp16.
// A thread's codes are contiguous in a page row (quad order for K, octet order
// for V), so both operands go from one coalesced global load per row straight
// into fragment registers, through a table indexed by a byte of codes: the
// half2 of a pair of 4-bit codes, or of pairs of 2-bit codes of two rows (6 bits of
// two 3-bit codes take a shift and a mask instead).  Copies for 32 lanes (16 of
// 8-byte entries, which are served in halves of a warp) leave no bank conflicts
// and make a row 128 bytes, so one dot product of the codes' word is the
// address.  V pairs join the codes of two tokens, interleaved by two masks per
// word.
// The running max moves only when a score passes it by kRoom (a vote; the
// shuffles and the rescale of 32 NT outputs run then: nearly every tile has a
// new max among its 16 rows, so moving it at once cost a fifth of the time).
// Value norms enter P' times a power of two that puts the largest one so far near
// kNorm (the same vote moves it), and a row of O is scaled by one of its own before
// its last rotation: fp16 ends at 2^-24, where the norms of a cache need not.
//
// q' = scale log2(e) q R^T comes ready from the launch that builds the work list
// (rotated in every segment it was most of a segment's set-up); out = O R runs on
// the same MMAs with O split into fp16 hi + lo, once per output row.
//
// Bound by the loop's shared-memory wavefronts (65 % of the SM's) and latency,
// 1.25 us a page and CTA; HBM would allow a fifth.  K4/V2, 8 KV heads of 128, g 4:
// 252 draft tokens over 256,960 156 us, 1.3 TB/s; K3/V3, g 5: 5 tokens over
// 131,001 140 us.  HP reads eight bytes a lookup and multiplies three times:
// 322 and 277 us.  168 registers are the most for three CTAs an SM; what the loop
// needs rarely is kept out of them where it would spill, which cost up to 25 us of the
// second.
#include "tq_internal.h"
#include "tq_ragged.cuh"

#include <limits.h>
#include <math.h>
#include <type_traits>

namespace tq {
namespace {

// A score may pass the running max by this much before the max moves: p <=
// 2^7, and with scaled value norms below 2^8 P' < 2^15 stays in fp16.
constexpr float kRoom = 7.f;
constexpr float kNorm = 256.f;
constexpr float kNoMax = -1e30f;   // below every score

struct FewParams {
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
  int Hkv, g, hc, nchunk, pcta;
  int Hq;
  int causal;
  uint32_t* status;
  RaggedAttend rg;
};

constexpr int kW = 4;                                       // warps: quarters of a page

// HP (fp16 and fp32 results): both operands of every product as fp16 hi + lo (hi hi
// + hi lo + lo hi, 22 bits).  A table entry then holds a pair's hi and lo.
template <int D, int KB, int VB, int NT, bool HP>
struct Few {
  static constexpr int NQ = 8 * NT;
  static constexpr bool KQ = KB == 2 && !HP, VQ = VB == 2 && !HP;   // two pairs per table entry
  // Which rarely needed values the loop holds is settled by its time at 168 registers (64
  // single tokens over 8,000 keys): with 8 rows each row's last key in registers (K3/V3
  // 181 us against 199 from shared memory, K2/V2 152 against 174, heads of 64 117
  // against 129); the first bad key noted at once for K4/V2 (162 us, kept to the end
  // 175), at the end for the others (K3/V3 181, at once 197; heads of 64 117, 134).
  static constexpr bool kLimits = NT == 1, kKeyNow = NT == 1 && D == 128 && KB == 4 && VB == 2;
  static constexpr int KT = 128 << (KQ ? 8 : 2 * KB), VT = 128 << (VQ ? 8 : 2 * VB);   // tables
  static constexpr int LDO = D + 4;                         // floats per row of an output (banks)
  static constexpr int LDA = D / 2 + 4;                     // words per row of a rotation operand
  // after the loop the table is dead: partial outputs, then the joined one and
  // the operand of the last rotation take its place
  static constexpr int OFF_P = 0;                           // [kW][NQ][LDO], the sum in the first
  static constexpr int OFF_ROT = (NQ * LDO * 4 + 127) & ~127;      // R fp16, over the other three
  static constexpr int OFF_A = tmax(OFF_ROT + 2 * D * D, kW * NQ * LDO * 4);   // [hi, lo][16][LDA]
  static constexpr int LOOP = KT + VT, END = OFF_A + 2 * 16 * LDA * 4;
  static constexpr int OFF_Q = LOOP > END ? LOOP : END;     // q' fp16 [NQ][D]
  static constexpr int OFF_M = OFF_Q + (HP ? 2 : 1) * 16 * D * 2;   // (HP: and lo); [kW][NQ] running max
  static constexpr int OFF_L = OFF_M + kW * NQ * 4;         // [kW][NQ] sums
  static constexpr int OFF_R = OFF_L + kW * NQ * 4;         // [16] sums, [16] maxima, flags
  static constexpr int BYTES = OFF_R + 256;
  static_assert(OFF_Q - OFF_A >= 8 * NQ * 16, "room for a batch of parts");
};

// N consecutive bytes of codes as little-endian words.  Multiples of 4 (and 2)
// are aligned loads; for other counts the words that hold them, shifted by `sh`
// when they are used: a prefetched value must not be touched before that.
template <int N>
struct Codes {
  static constexpr bool kOdd = N % 4 != 0 && N != 2;
  static constexpr int NW = (N + 3) / 4, NR = kOdd ? 2 : NW;
  uint32_t raw[NR];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (N == 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
    } else if constexpr (N == 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      raw[0] = v.x; raw[1] = v.y;
    } else if constexpr (N == 2) {
      raw[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
    } else {
      // 3 or 6 bytes: two words (the second may lie past the row, but within
      // the page: norms follow the codes)
#pragma unroll
      for (int i = 0; i < NR; ++i) raw[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    }
  }
  __device__ __forceinline__ void words(uint32_t (&w)[NW], uint32_t sh) const {
    if constexpr (kOdd) {
      w[0] = __funnelshift_r(raw[0], raw[1], sh);
      if constexpr (NW > 1) w[1] = raw[1] >> sh;
    } else {
#pragma unroll
      for (int i = 0; i < NW; ++i) w[i] = raw[i];
    }
  }
};

// Aligned start and shift of N bytes at offset `off`.
template <int N>
__device__ __forceinline__ int code_start(int off, uint32_t& sh) {
  constexpr bool odd = N % 4 != 0 && N != 2;
  sh = odd ? (uint32_t)(off & 3) * 8 : 0;
  return odd ? off & ~3 : off;
}

// Shared address of the table row of field `k` (FB bits each, low first) of the
// words: base + 128 field.  A byte takes one dot product with 128 in its place.
template <int FB, int NW>
__device__ __forceinline__ uint32_t field_at(const uint32_t (&w)[NW], int k, uint32_t base) {
  const int bo = FB * k, wi = bo >> 5, sh = bo & 31;
  if constexpr (FB == 8) {
    return __dp4a(w[wi], 128u << sh, base);
  } else {
    constexpr uint32_t mask = ((1u << FB) - 1u) << 7;
    uint32_t x;
    if (sh + FB > 32) x = __funnelshift_r(w[wi], w[wi + 1 < NW ? wi + 1 : wi], sh) << 7;
    else if (sh >= 7) x = w[wi] >> (sh - 7);
    else x = w[wi] << (7 - sh);
    return (x & mask) + base;
  }
}

// volatile: not to be moved over the barriers around the table's lifetime
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t& x, uint32_t& y) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(addr));
}

// HP: field k of x and of y, hi and lo.
template <int FB, int NW>
__device__ __forceinline__ void look_up_split(uint32_t base, const uint32_t (&x)[NW],
                                              const uint32_t (&y)[NW], int k, uint32_t& h0,
                                              uint32_t& h1, uint32_t& l0, uint32_t& l1) {
  lds64(field_at<FB>(x, k, base), h0, l0);
  lds64(field_at<FB>(y, k, base), h1, l1);
}

// One pair of each of two rows (registers a0 and a1, or a2 and a3, of an A
// fragment): field k of x and of y, or, with quad entries, byte k of x.
template <int FB, bool Q, int NW>
__device__ __forceinline__ void look_up2(uint32_t base, const uint32_t (&x)[NW],
                                         const uint32_t (&y)[NW], int k, uint32_t& r0,
                                         uint32_t& r1) {
  if constexpr (Q) {
    // bytes of even fields lie in x, of odd fields in y (join_nibbles)
    lds64((k & 1) ? field_at<8>(y, k >> 1, base) : field_at<8>(x, k >> 1, base), r0, r1);
  } else {
    r0 = lds32(field_at<FB>(x, k, base));
    r1 = lds32(field_at<FB>(y, k, base));
  }
}

// Nibbles of x (low) and y (high) joined into bytes: even ones into x, odd into y.
template <int NW>
__device__ __forceinline__ void join_nibbles(uint32_t (&x)[NW], uint32_t (&y)[NW]) {
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint32_t e = (x[i] & 0x0F0F0F0Fu) | ((y[i] << 4) & 0xF0F0F0F0u);
    y[i] = ((x[i] >> 4) & 0x0F0F0F0Fu) | (y[i] & 0xF0F0F0F0u);
    x[i] = e;
  }
}

__device__ __forceinline__ const uint8_t* page_at(const uint8_t* base, int e, int page_bytes) {
  const uint8_t* r;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(r) : "r"(e), "r"(page_bytes), "l"(base));
  return r;
}

// Fields of two tokens' VB-bit codes joined into pairs: even entries in e, odd
// ones in o (2 VB bits each, entry 2 k (+ 1) at field k).
template <int VB, int NW>
__device__ __forceinline__ void join_tokens(const uint32_t (&a)[NW], const uint32_t (&b)[NW],
                                            uint32_t (&e)[NW], uint32_t (&o)[NW]) {
  // VB bits of every 2 VB, continued across the words
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < 32; ++t)
      if ((((32 * i + t) / VB) & 1) == 0) m |= 1u << t;
    const uint32_t am = a[i] & m;
    uint32_t bl = b[i] << VB;                              // b's even codes up by VB
    if (i > 0) bl = __funnelshift_l(b[i - 1], b[i], VB);
    e[i] = am | (bl & ~m);
    uint32_t ar = a[i] >> VB;                              // a's odd codes down by VB
    if (i + 1 < NW) ar = __funnelshift_r(a[i], a[i + 1], VB);
    o[i] = (ar & m) | (b[i] & ~m);
  }
}

template <int D, int KB, int VB>
struct FewTile {
  static constexpr int KN = D / 4 * KB / 8, VN = D / 8 * VB / 8;
  Codes<KN> k[2];               // tokens gq, gq + 8: quad tq
  Codes<VN> v[4];               // tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9: octet gq
  uint16_t kn[2], vn[2];        // fp16 norms of tokens gq, gq + 8
};

// fp16 hi + lo of a pair (2^-22 of each value)
__device__ __forceinline__ uint32_t split2(float a, float b, uint32_t& lo) {
  const uint32_t hi = pack_half2(a, b);
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  lo = pack_half2(a - __low2float(h), b - __high2float(h));
  return hi;
}

// B fragment (16 deep, 8 wide) of R[j][i], j = 16 ch + .. deep, i = 8 jt + .. wide,
// from R's fp16 rows in shared memory, their 16-byte pieces moved by row (r7).
template <int D>
__device__ __forceinline__ void frag_of_rotation(uint32_t (&b)[2], const unsigned char* r, int ch,
                                                 int jt, int lane) {
  const int row = 16 * ch + (lane & 15);
  const unsigned char* at = r + row * (2 * D) + ((jt ^ (row & 7)) << 4);
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];"
               : "=r"(b[0]), "=r"(b[1]) : "r"(smem_u32(at)));
}

// c += O R of 8 columns (8 jt ..): O's hi words, and its lo where LO.
template <int D, bool LO>
__device__ __forceinline__ void rotate_slice(float (&c)[4], const unsigned char* rot,
                                             const uint32_t* A, int jt, int lane) {
  constexpr int LDA = D / 2 + 4;
  const int gq = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int ch = 0; ch < D / 16; ++ch) {
    uint32_t r[2], ah[4], al[4];
    frag_of_rotation<D>(r, rot, ch, jt, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (gq + 8 * (i & 1)) * LDA + 8 * ch + tq + 4 * (i >> 1);
      ah[i] = A[at];
      if (LO) al[i] = A[16 * LDA + at];
    }
    mma_f16_16816(c, ah, r[0], r[1]);
    if (LO) mma_f16_16816(c, al, r[0], r[1]);
  }
}

// A table of 128-byte rows from a codebook.
template <int BITS, bool Q, bool HP>
__device__ __forceinline__ void fill_table(unsigned char* table, const float* cent, int tid,
                                           int nthreads) {
  constexpr int N = 1 << (Q ? 4 * BITS : 2 * BITS);
  constexpr uint32_t M = (1u << BITS) - 1u;
  for (int i = tid; i < 8 * N; i += nthreads) {
    const uint32_t e = (uint32_t)i >> 3;
    uint32_t lo;
    const uint32_t x = split2(__ldg(cent + (e & M)), __ldg(cent + ((e >> BITS) & M)), lo);
    const uint32_t y = HP ? lo : Q ? pack_half2(__ldg(cent + ((e >> (2 * BITS)) & M)),
                                      __ldg(cent + ((e >> (3 * BITS)) & M))) : x;
    reinterpret_cast<uint4*>(table + e * 128)[i & 7] = make_uint4(x, y, x, y);
  }
}

template <int D, int KB, int VB, int NT, bool HP>
__device__ __forceinline__ void fill_tables(const FewParams& p, unsigned char* sm) {
  using F = Few<D, KB, VB, NT, HP>;
  fill_table<KB, F::KQ, HP>(sm, p.kc, threadIdx.x, 32 * kW);
  fill_table<VB, F::VQ, HP>(sm + F::KT, p.vc, threadIdx.x, 32 * kW);
}

// One segment of the work list.
template <int D, int KB, int VB, int NT, bool HP>
__device__ __forceinline__ void attend_segment(const FewParams& p, const SegWork& sw,
                                               unsigned char* sm, bool filled) {
  using F = Few<D, KB, VB, NT, HP>;
  using Tile = FewTile<D, KB, VB>;
  constexpr int NQ = F::NQ, NC = D / 16, kThreads = 32 * kW, LDA = F::LDA, LDO = F::LDO;
  constexpr int KROW = D * KB / 8, VROW = D * VB / 8;
  float* mw = reinterpret_cast<float*>(sm + F::OFF_M);
  float* lw = reinterpret_cast<float*>(sm + F::OFF_L);
  float* U = reinterpret_cast<float*>(sm + F::OFF_P);
  uint32_t* A = reinterpret_cast<uint32_t*>(sm + F::OFF_A);
  float* rowl = reinterpret_cast<float*>(sm + F::OFF_R);
  int* flags = reinterpret_cast<int*>(sm + F::OFF_R + 128);   // last CTA, first bad key
  int* lims = reinterpret_cast<int*>(sm + F::OFF_R + 192);    // [NQ] last key each row sees

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  const int kvh = sw.group / p.nchunk, chunk = sw.group % p.nchunk;
  const int h0 = kvh * p.g + chunk * p.hc;                 // first query head
  const int nh = min(p.hc, p.g - chunk * p.hc);            // heads of this CTA
  const int64_t stream = (int64_t)sw.seg.req * p.Hkv + kvh;
  const int q_len = (int)sw.rq.q_len, pos0 = sw.seg.tile * p.pcta;
  // keys in the pages, position of the request's row 0: 32 bits (base + q_len is a length)
  const int seq = (int)sw.rq.seq, t_base = (int)sw.rq.base;
  // row n of the CTA: position pos0 + n / hc, head h0 + n % hc
  auto row_pos = [&](int n) { return n < p.pcta * p.hc ? pos0 + n / p.hc : INT_MAX; };
  auto row_valid = [&](int n) { return row_pos(n) < q_len && n % p.hc < nh; };
  auto row_at = [&](int n, const int64_t (&s)[3]) {
    return (sw.rq.q0 + row_pos(n)) * s[1] + (int64_t)(h0 + n % p.hc) * s[0];
  };
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
  const int32_t* bt = p.pm.bt ? p.pm.bt + stream * p.pm.bt_stride : nullptr;
  const int slot0 = (int)(stream * p.pm.pps);              // contiguous layout
  auto entry = [&](int pg) -> int {
    pg = min(pg, pend - 1);
    return bt ? __ldg(bt + pg) : slot0 + pg;
  };
  auto load_tile = [&](Tile& x, int e) {
    if ((unsigned)e >= (unsigned)p.nblocks) {              // e < 0 too
      atomicOr(p.status, TQ_DEV_BAD_BLOCK);
      e = 0;
    }
    // 16 rows of 128: one product, since three addresses across the loop cost spills;
    // elsewhere, where there are registers, three (encoder 35.0 us against 36.0)
    const uint8_t *k, *v, *n;
    if constexpr (D * NT <= 128) {
      k = page_at(p.pages + at_k, e, p.page_bytes);
      v = page_at(p.pages + at_v, e, p.page_bytes);
      n = page_at(p.pages + at_n, e, p.page_bytes);
    } else {
      const uint8_t* page = page_at(p.pages, e, p.page_bytes);
      k = page + at_k;
      v = page + at_v;
      n = page + at_n;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.k[i].load(k + 8 * i * KROW);
      x.kn[i] = __ldg(reinterpret_cast<const uint16_t*>(n + 16 * i));
      x.vn[i] = __ldg(reinterpret_cast<const uint16_t*>(n + 128 + 16 * i));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i].load(v + ((i & 1) + 8 * (i >> 1)) * VROW);
  };
  int pg = sw.seg.kt0;
  const bool any = pg < pend;
  Tile cur, nxt;
  int e_next = 0, e_after = 0;
  if (any) {
    e_next = entry(pg + 1);
    e_after = entry(pg + 2);
    load_tile(cur, entry(pg));
  }

  // ---- query rows, table ---------------------------------------------------------
  if (tid == 0) flags[1] = INT_MAX;
  if (tid < NQ) lims[tid] = row_lim(tid);
  // 16-byte piece k of row n, quad t of q' (quad order): its place in the row
  auto q_piece = [](int n, int t, int k) {
    const int f = D == 128 ? ((t >> 1) | ((n & 1) << 1)) : (n & 1);
    return n * (D / 8) + t * (D / 32) + (k ^ f);
  };
  const int64_t tok0 = p.qp_stride ? sw.seg.req * p.qp_stride : sw.rq.q0;
  constexpr int kQLo = 16 * D * 2;                         // HP: lo behind hi
#pragma unroll
  for (int part = 0; part < (HP ? 2 : 1); ++part)
    for (int i = tid; i < NQ * D / 8; i += kThreads) {
      const int n = i / (D / 8), c = i % (D / 8);
      unsigned char* dst = sm + F::OFF_Q + part * kQLo + 16 * q_piece(n, c / (D / 32), c % (D / 32));
      if (row_valid(n))
        cp_async16(dst, p.qp + ((tok0 + row_pos(n)) * p.Hq + h0 + n % p.hc) * (HP ? 2 * D : D) +
                            part * D + 8 * c);
      else
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
    }
  if (!filled) fill_tables<D, KB, VB, NT, HP>(p, sm);
  cp_async_wait_all();
  __syncthreads();

  // ---- pages -----------------------------------------------------------------------
  float O[NC][NT][4];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) O[i][n][0] = O[i][n][1] = O[i][n][2] = O[i][n][3] = 0.f;
  // m: what scores are taken relative to; finite from the start, so a row
  // without keys needs no case of its own
  float m[NT][2], l[NT][2];
  float vs = 4194304.f;                                    // scale of the value norms, 2^22 at most
  int lim_min = INT_MAX, lim[2] = {INT_MAX, INT_MAX};
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = kNoMax;
      l[n][c] = 0.f;
      if (F::kLimits) lim[c] = lims[2 * tq + c];
      lim_min = min(lim_min, lims[8 * n + 2 * tq + c]);
    }
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
  lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));
  const uint32_t k_base = smem_u32(sm) + (F::KQ || HP ? 8 * (lane & 15) : 4 * lane);
  const uint32_t v_base = smem_u32(sm + F::KT) + (F::VQ || HP ? 8 * (lane & 15) : 4 * lane);

  int bad_key = INT_MAX;

  // one page: `cur` is used, `nxt` takes the next page's codes
  auto step = [&](Tile& cur, Tile& nxt) {
    load_tile(nxt, e_next);
    e_next = e_after;
    if (warp == 0 && lane == 0 && (unsigned)e_after < (unsigned)p.nblocks)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                   ::"l"(page_at(p.pages, e_after, p.page_bytes)), "r"(p.page_bytes) : "memory");
    e_after = entry(pg + 3);
    const int key0 = 64 * pg + s0 + gq;
    float kn[2], vn[2], s[NT][4];
    // norms: 0 past the end; a token whose norm is not finite counts as 0 (0 x
    // inf would reach rows that do not see it) and the rows that see it become
    // NaN at the end
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h = (uint32_t)cur.kn[i] | ((uint32_t)cur.vn[i] << 16);
      const bool in = key0 + 8 * i < kend;
      // exponent 31 in either half carries into its sign bit
      const bool fin = (((h & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u) == 0;
      if (in && !fin) {
        if constexpr (F::kKeyNow) atomicMin(&flags[1], key0 + 8 * i);
        else bad_key = min(bad_key, key0 + 8 * i);
      }
      h = in && fin ? h : 0u;
      const __half2 h2 = *reinterpret_cast<const __half2*>(&h);
      kn[i] = __low2float(h2);
      vn[i] = __high2float(h2) * vs;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    uint32_t kw[2][Codes<Tile::KN>::NW];
    cur.k[0].words(kw[0], ksh);
    cur.k[1].words(kw[1], ksh);
    if (F::KQ) join_nibbles(kw[0], kw[1]);
    // S^T: two chunks of 16 dims share one 16-byte piece of q'
#pragma unroll
    for (int c2 = 0; c2 < NC / 2; ++c2) {
      uint4 qb[NT], ql[HP ? NT : 1];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const unsigned char* at = sm + F::OFF_Q + 16 * q_piece(8 * n + gq, tq, c2);
        qb[n] = *reinterpret_cast<const uint4*>(at);
        if constexpr (HP) ql[n] = *reinterpret_cast<const uint4*>(at + kQLo);
      }
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
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16_16816(s[n], a, c ? qb[n].z : qb[n].x, c ? qb[n].w : qb[n].y);
          if constexpr (HP) {
            mma_f16_16816(s[n], a, c ? ql[n].z : ql[n].x, c ? ql[n].w : ql[n].y);
            mma_f16_16816(s[n], al, c ? qb[n].z : qb[n].x, c ? qb[n].w : qb[n].y);
          }
        }
      }
    }
    // relative to m
    float d[NT][4], top = -INFINITY;
    const bool edge = 64 * pg + s0 + 15 > lim_min;
    // key i of the tile hidden from column c of slice n
    auto hidden = [&](int n, int i, int c) { return key0 + 8 * i > (F::kLimits ? lim[c] : lims[8 * n + 2 * tq + c]); };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[n][i] = fmaf(s[n][i], kn[i >> 1], -m[n][i & 1]);
    if (edge) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hidden(n, i >> 1, i & 1)) d[n][i] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) top = fmaxf(fmaxf(fmaxf(top, d[n][0]), fmaxf(d[n][1], d[n][2])), d[n][3]);
    const float big = fmaxf(fabsf(vn[0]), fabsf(vn[1]));
    if (__any_sync(0xffffffffu, top > kRoom || big >= kNorm)) {
      // the largest norm of the tile, below 2^(e + 1): down to below kNorm
      const int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23) - 127;
      const float r = __uint_as_float((uint32_t)(127 - max(e - 7, 0)) << 23);
      vs *= r;
      vn[0] *= r;
      vn[1] *= r;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // the largest score of the column in this tile
          const bool out0 = edge && hidden(n, 0, c), out1 = edge && hidden(n, 1, c);
          float x = fmaxf(out0 ? -INFINITY : s[n][c] * kn[0], out1 ? -INFINITY : s[n][2 + c] * kn[1]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float mn = fmaxf(m[n][c], x), f = fast_exp2(m[n][c] - mn);
          l[n][c] *= f;
#pragma unroll
          for (int i = 0; i < NC; ++i) { O[i][n][c] *= f * r; O[i][n][2 + c] *= f * r; }
          m[n][c] = mn;
          d[n][c] = out0 ? -INFINITY : fmaf(s[n][c], kn[0], -mn);
          d[n][2 + c] = out1 ? -INFINITY : fmaf(s[n][2 + c], kn[1], -mn);
        }
    }
    uint32_t pb[NT][2], pl[HP ? NT : 1][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = fast_exp2(d[n][2 * i]), p1 = fast_exp2(d[n][2 * i + 1]);
        l[n][0] += p0;
        l[n][1] += p1;
        if constexpr (HP) {
          uint32_t lo;
          pb[n][i] = movmatrix_trans(split2(p0 * vn[i], p1 * vn[i], lo));
          pl[n][i] = movmatrix_trans(lo);
        } else {
          pb[n][i] = movmatrix_trans(pack_half2(p0 * vn[i], p1 * vn[i]));
        }
      }
    }
    constexpr int VW = Codes<Tile::VN>::NW;
    uint32_t ve[2][VW], vo[2][VW];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t x[VW], y[VW];
      cur.v[2 * i].words(x, vsh);
      cur.v[2 * i + 1].words(y, vsh);
      join_tokens<VB>(x, y, ve[i], vo[i]);
      if (F::VQ) join_nibbles(ve[i], vo[i]);
    }
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
      for (int n = 0; n < NT; ++n) {
        mma_f16_16816(O[c][n], a, pb[n][0], pb[n][1]);
        if constexpr (HP) {
          mma_f16_16816(O[c][n], a, pl[n][0], pl[n][1]);
          mma_f16_16816(O[c][n], al, pb[n][0], pb[n][1]);
        }
      }
    }
  };
#pragma unroll 1
  while (pg < pend) {                                      // by twos: no copies between tiles
    step(cur, nxt);
    if (++pg >= pend) break;
    step(nxt, cur);
    ++pg;
  }

  if (bad_key != INT_MAX) atomicMin(&flags[1], bad_key);

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
  __syncthreads();                                         // and the table is dead
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = 8 * n + 2 * tq + c;
      float M = mw[col];
#pragma unroll
      for (int w = 1; w < kW; ++w) M = fmaxf(M, mw[w * NQ + col]);
      // times 1 / vs (exponents: vs is a power of two)
      const float f = fast_exp2(m[n][c] - M) * __uint_as_float(0x7F000000u - __float_as_uint(vs));
      float* mine = U + (warp * NQ + col) * LDO + gq;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        mine[16 * i] = O[i][n][c] * f;
        mine[16 * i + 8] = O[i][n][2 + c] * f;
      }
    }
  if (tid < NQ) {
    float M = mw[tid], x = 0.f;
#pragma unroll
    for (int w = 1; w < kW; ++w) M = fmaxf(M, mw[w * NQ + tid]);
#pragma unroll
    for (int w = 0; w < kW; ++w) x += lw[w * NQ + tid] * fast_exp2(mw[w * NQ + tid] - M);
    if (flags[1] <= row_lim(tid)) x = NAN;
    rowl[tid] = x;
    rowl[16 + tid] = M;
  }
  __syncthreads();
  for (int i = tid; i < NQ * D / 4; i += kThreads) {
    const int n = i / (D / 4), at = n * LDO + 4 * (i % (D / 4));
    float4 x = *reinterpret_cast<const float4*>(U + at);
#pragma unroll
    for (int w = 1; w < kW; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(U + w * NQ * LDO + at);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    *reinterpret_cast<float4*>(U + at) = x;
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
        const float2 x = __ldg(reinterpret_cast<const float2*>(p.rot + 8 * i) + e);
        split2(x.x, x.y, w[e]);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      cp_async16(dst, p.rot_h + 8 * i);
    }
  }

  // ---- a split tile: partials out, the last CTA joins them -----------------------
  if (sw.seg.slot >= 0) {
    const RaggedPlan& pl = p.rg.plan;
    for (int i = tid; i < NQ * D / 4; i += kThreads) {
      const int n = i / (D / 4), at = 4 * (i % (D / 4));
      if (row_valid(n))
        *reinterpret_cast<float4*>(pl.part + part_row(pl, sw.seg.slot, sw.group, n) * D + at) =
            *reinterpret_cast<const float4*>(U + n * LDO + at);
    }
    if (tid < NQ) pl.ml[part_row(pl, sw.seg.slot, sw.group, tid)] = make_float2(rowl[16 + tid], rowl[tid]);
    if (!last_of_tile(pl, sw, &flags[0])) {
      cp_async_wait_all();                                 // nothing in flight into what comes next
      return;
    }
    // every part's {m, l} in one trip, then the weights 2^(m - M); parts come in
    // slot order whatever the order of arrival
    const int parts = sw.seg.parts;
    float2* wl = reinterpret_cast<float2*>(sm + F::OFF_A);   // [parts][NQ] of a batch of parts
    constexpr int kBatch = (F::OFF_Q - F::OFF_A) / (8 * NQ);
    constexpr int NE = NQ * D / 4 / kThreads;              // float4 columns per thread
    float4 acc[NE];
    const float* src[NE];                                  // the first part's values, or NULL
    const int64_t next_part = (int64_t)pl.G * pl.rows * D;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int i = tid + k * kThreads, n = i / (D / 4);
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      src[k] = row_valid(n) ? pl.part + part_row(pl, sw.seg.first, sw.group, n) * D + 4 * (i % (D / 4))
                            : nullptr;
    }
    float run_m = kNoMax, run_l = 0.f;                     // of row tid (tid < NQ)
    for (int s0 = 0; s0 < parts; s0 += kBatch) {
      const int ns = min(kBatch, parts - s0);
      for (int i = tid; i < ns * NQ; i += kThreads)
        wl[i] = __ldcg(pl.ml + part_row(pl, sw.seg.first + s0 + i / NQ, sw.group, i % NQ));
      __syncthreads();
      if (tid < NQ) {
        float M = run_m;
        for (int s = 0; s < ns; ++s) M = fmaxf(M, wl[s * NQ + tid].x);
        const float f = fast_exp2(run_m - M);              // of what earlier batches left
        run_l *= f;
        for (int s = 0; s < ns; ++s) {
          const float w = fast_exp2(wl[s * NQ + tid].x - M);
          run_l = fmaf(w, wl[s * NQ + tid].y, run_l);
          wl[s * NQ + tid].x = w;
        }
        run_m = M;
        rowl[tid] = f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NE; ++k) {
        const int n = (tid + k * kThreads) / (D / 4);
        const float f = rowl[n];
        acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
      }
#pragma unroll 4
      for (int s = 0; s < ns; ++s) {
#pragma unroll
        for (int k = 0; k < NE; ++k) {
          if (!src[k]) continue;
          const float4 x = __ldcg(reinterpret_cast<const float4*>(src[k] + s * next_part));
          const float w = wl[s * NQ + (tid + k * kThreads) / (D / 4)].x;
          acc[k].x = fmaf(w, x.x, acc[k].x);
          acc[k].y = fmaf(w, x.y, acc[k].y);
          acc[k].z = fmaf(w, x.z, acc[k].z);
          acc[k].w = fmaf(w, x.w, acc[k].w);
        }
      }
#pragma unroll
      for (int k = 0; k < NE; ++k)
        if (src[k]) src[k] += ns * next_part;
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int i = tid + k * kThreads;
      *reinterpret_cast<float4*>(U + i / (D / 4) * LDO + 4 * (i % (D / 4))) = acc[k];
    }
    if (tid < NQ) rowl[tid] = run_l;
    __syncthreads();
  }

  // ---- out = (O / l) R ---------------------------------------------------------------
  // a warp per row: O / l times the power of two that puts its largest value into
  // [2^10, 2^11), which the result is divided by
#pragma unroll
  for (int n0 = 0; n0 < 16; n0 += kW) {
    const int n = n0 + warp;
    float2 u[D / 64];
    float top = 0.f;
    const bool valid = n < NQ && row_valid(n);
    const float x = valid ? rowl[n] : 0.f, il = x == 0.f ? 0.f : 1.f / x;
#pragma unroll
    for (int k = 0; k < D / 64; ++k) {
      u[k] = make_float2(0.f, 0.f);
      if (valid) u[k] = *reinterpret_cast<const float2*>(U + n * LDO + 2 * (lane + 32 * k));
      u[k].x *= il;
      u[k].y *= il;
      top = fmaxf(top, fmaxf(fabsf(u[k].x), fabsf(u[k].y)));
    }
    // (a row of NaN has none: the maximum leaves NaN out; of zeros neither)
    const int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
    const int up = e == 128 ? 0 : min(10 - e, 100);
    const float s = __uint_as_float((uint32_t)(127 + up) << 23);
    if (lane == 0) rowl[16 + n] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int k = 0; k < D / 64; ++k) {
      const int w = lane + 32 * k;
      A[n * LDA + w] = split2(u[k].x * s, u[k].y * s, A[(16 + n) * LDA + w]);
    }
  }
  cp_async_wait_all();
  __syncthreads();
  int64_t o_at[2];
  bool o_ok[2];
  float o_inv[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int n = gq + 8 * r;
    o_ok[r] = n < NQ && row_valid(n);
    o_at[r] = o_ok[r] ? row_at(n, p.os) : 0;
    o_inv[r] = rowl[16 + n];
  }
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
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (!o_ok[r]) continue;
      const int64_t o = o_at[r] + (int64_t)(8 * jt + 2 * tq) * p.os[2];
      const float x = c[2 * r] * o_inv[r], y = c[2 * r + 1] * o_inv[r];
      if (p.o_pair) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        reinterpret_cast<uint32_t*>(p.out)[o >> 1] =
            p.o_dtype == TQ_BF16 ? *reinterpret_cast<const uint32_t*>(&h) : pack_half2(x, y);
      } else {
        store_elem(p.out, p.o_dtype, o, x);
        store_elem(p.out, p.o_dtype, o + p.os[2], y);
      }
    }
  }
}

template <int D, int KB, int VB, int NT, bool HP>
__global__ void __launch_bounds__(32 * kW, HP && D * NT == 256 ? 2 : 3) attend_few_kernel(FewParams p) {
  extern __shared__ __align__(128) unsigned char sm[];
  // segments in the list's order (long ones first), whoever is free next
  __shared__ int next;
  bool filled = true;
  fill_tables<D, KB, VB, NT, HP>(p, sm);                   // beside the launch before
  pdl_wait();                                              // the list and q'
  for (;; filled = false) {
    __syncthreads();                                       // the last segment is done with
    if (threadIdx.x == 0) next = atomicAdd(p.rg.plan.next, 1);
    __syncthreads();
    SegWork sw;
    if (!take_segment(p.rg, next, sw)) return;
    attend_segment<D, KB, VB, NT, HP>(p, sw, sm, filled);
  }
}
using FewFn = void (*)(FewParams);

template <int D, int NT, bool HP>
FewFn few_fn(int kb, int vb, int& bytes) {
#define TQ_FEW(K, V) \
  if (kb == K && vb == V) { bytes = Few<D, K, V, NT, HP>::BYTES; return attend_few_kernel<D, K, V, NT, HP>; }
  TQ_FEW(4, 2) TQ_FEW(4, 3) TQ_FEW(4, 4) TQ_FEW(3, 2) TQ_FEW(3, 3) TQ_FEW(3, 4)
  TQ_FEW(2, 2) TQ_FEW(2, 3) TQ_FEW(2, 4)
#undef TQ_FEW
  return nullptr;
}

}  // namespace

bool attend_few_applies(const tq_geom* G) {
  int bytes;
  if (G->head_dim == 128) return few_fn<128, 1, false>(G->key_bits, G->value_bits, bytes) != nullptr;
  if (G->head_dim == 64) return few_fn<64, 1, false>(G->key_bits, G->value_bits, bytes) != nullptr;
  return false;
}

int launch_attend_few(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                      const tq_attend_args* a, const RaggedAttend& rg, int64_t Hkv, int hc,
                      int pcta, int rows, const __half* qp, int64_t qp_stride, int64_t grid,
                      uint32_t* status, cudaStream_t st) {
  FewParams p;
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
  p.Hkv = (int)Hkv;
  p.g = (int)(a->q->shape[1] / Hkv);
  p.hc = hc;
  p.nchunk = (p.g + hc - 1) / hc;
  p.pcta = pcta;
  p.causal = a->causal;
  p.status = status;
  p.rg = rg;
  FewFn fn;
  int bytes = 0;
  auto pick = [&](auto d, auto nt) {
    constexpr int D = decltype(d)::value, NT = decltype(nt)::value;
    fn = attend_precise(a) ? few_fn<D, NT, true>(G->key_bits, G->value_bits, bytes)
                           : few_fn<D, NT, false>(G->key_bits, G->value_bits, bytes);
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  if (G->head_dim == 128) {
    if (rows == 8) pick(std::integral_constant<int, 128>(), I1()); else pick(std::integral_constant<int, 128>(), I2());
  } else {
    if (rows == 8) pick(std::integral_constant<int, 64>(), I1()); else pick(std::integral_constant<int, 64>(), I2());
  }
  if (set_smem_attr((const void*)fn, bytes) != TQ_OK) return TQ_ERR_CUDA;
  // CTAs that fit at once
  const int64_t fit = (int64_t)device_sm_count() * occupancy((const void*)fn, 32 * kW, bytes);
  return launch_result(launch_pdl(fn, dim3((unsigned)tmin(grid, fit)), dim3(32 * kW), bytes, st, p),
                       "tq_attend_ragged/few");
}

}  // namespace tq
