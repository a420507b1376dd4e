// tq_attend_few.cuh — what the few-row attention kernels share (tq_attend_few.cu: one
// softmax map; tq_attend_pair.cu: two maps of keys of their own): codes from global
// memory into mma.sync fragments through lane-replicated tables, and the rotation of
// the output rows.
#pragma once

#include "tq_common.cuh"
#include "tq_ragged.cuh"

namespace tq {
namespace few {

// A score may pass the running max by this much before the max moves: p <=
// 2^7, and with scaled value norms below 2^8 P' < 2^15 stays in fp16.
constexpr float kRoom = 7.f;
constexpr float kNorm = 256.f;
constexpr float kNoMax = -1e30f;   // below every score

constexpr int kW = 4;              // warps of a CTA: quarters of a page

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

}  // namespace few
}  // namespace tq
