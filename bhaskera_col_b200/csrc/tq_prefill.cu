// tq_prefill.cu — causal (or full) attention of a chunk of queries straight
// off the packed TurboQuant pages: the prefill attention of a layer.
//
// Replaces: HF attention (torch SDPA, causal, GQA repeat) over the
// dequantised K/V that TurboQuantKVCache.update returns during prefill
// (kv_cache.py:445-490 -> 483-488; engine.py:389).  The keys and values it
// attends are the reference's dequantised ones, x^ = n (c[idx] R): the MSE
// codes only (a QJL sketch, when the cache keeps one, refines decode scores
// and is not used here).
//
// Math, as in the decode kernel: <q, k_t> = n_t <q R^T, c_k[idx_t]> and
// sum_t p_t v_t = (sum_t p_t n_t c_v[idx_t]) R, so each CTA rotates its
// queries once, attends centroid values decoded from the codes, and
// un-rotates its output once.
//
// One CTA = 128 query rows of one KV head's GQA group: hc heads (the largest
// of 8, 4, 2, 1 dividing the group) x 128 / hc consecutive positions, 8 warps
// of 16 rows, so each decoded page serves hc heads.  Per 64-token page (one key tile): a bulk async copy brings the
// page into shared memory (double-buffered, mbarrier), all threads decode the
// K and V codes into fp16 tiles in coordinate order, then every warp runs
// S = Q' K^T and O += P' V with mma.sync m16n8k16 (fp16 in, fp32 accumulate)
// and an online softmax; P' = P * ||v|| folds the value norms in.
#include "tq_common.cuh"
#include "tq_internal.h"
#include "tq_ragged.cuh"

#include <limits.h>
#include <math.h>
#include <type_traits>

namespace tq {
namespace {

constexpr int kPfWarps = 8;
constexpr int kPfThreads = 32 * kPfWarps;
constexpr float kLog2eP = 1.4426950408889634f;

struct PrefillParams {
  const uint8_t* pages;
  PageMap pm;
  int page_bytes, page_pitch, off_v, off_kn, off_vn;   // page geometry (make_geom)
  const __half* rot_h;          // R [D][D] fp16, row-major
  const float* rot;             // R [D][D] (HP kernels)
  const float* kc;
  const float* vc;
  const void* q; int q_dtype; int64_t qs[4];     // (B, Hq, Tq, D)
  void* out; int o_dtype; int64_t os[4];
  int64_t Hq, Hkv, g, Tq, n_tokens;
  int hc;                       // query heads per CTA
  float scale;                  // softmax scale
  int causal;
  int nqb;                      // query blocks per head
  const int32_t* kv_start;      // [B] first attended key of each batch row, or NULL
  uint32_t* status;
  RaggedAttend rg;              // ragged batch (RG kernels): Tq, n_tokens come per request
};

// HP: the products take both operands as fp16 hi + lo (hi hi + lo hi + hi lo, 22
// bits): R, the centroids, the queries and the probabilities.
template <int D, int KB, int VB, bool HP>
struct Pf {
  static constexpr int KROW = D * KB / 8, VROW = D * VB / 8;
  static constexpr int LD = D + 8;                          // padded fp16 row (ldmatrix)
  static constexpr int OFF_R = 0;
  static constexpr int OFF_KS = OFF_R + D * LD * 2;
  static constexpr int OFF_VS = OFF_KS + 64 * LD * 2;
  static constexpr int OFF_NRM = OFF_VS + 64 * LD * 2;     // kn[64], vn[64] floats
  static constexpr int OFF_LUT = OFF_NRM + 512;            // K, V fp16 tables (256 each)
  static constexpr int OFF_BAR = OFF_LUT + 1024;
  static constexpr int OFF_LO = OFF_BAR + 128;             // HP: R, K, V and the tables, lo
  static constexpr int LO_K = D * LD, LO_V = LO_K + 64 * LD, LO_LUT = LO_V + 64 * LD;   // halves
  static constexpr int OFF_STG = OFF_LO + (HP ? LO_LUT * 2 + 1024 : 0);   // 2 page stages (runtime size)
  static int smem(int page_pitch) { return OFF_STG + 2 * page_pitch; }
};

// fp16 hi of a pair, and lo (2^-22 of each value in both)
__device__ __forceinline__ uint32_t split_half2(float a, float b, uint32_t& lo) {
  const uint32_t hi = pack_half2(a, b);
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  lo = pack_half2(a - __low2float(h), b - __high2float(h));
  return hi;
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}

// B fragments of two n-tiles (n0..n0+15) for k-chunk k0..k0+15 from a tile
// stored [n][k] (k contiguous, row stride ld halves).
__device__ __forceinline__ void frag_b_nk(uint32_t (&r)[4], const __half* base, int ld, int n0,
                                          int k0, int lane) {
  const int row = n0 + (lane & 7) + ((lane >> 4) << 3);
  const int col = k0 + (((lane >> 3) & 1) << 3);
  ldsm_x4(r, base + row * ld + col);
}
// Same from a tile stored [k][n] (n contiguous).
__device__ __forceinline__ void frag_b_kn(uint32_t (&r)[4], const __half* base, int ld, int n0,
                                          int k0, int lane) {
  const int row = k0 + (lane & 7) + (((lane >> 3) & 1) << 3);
  const int col = n0 + ((lane >> 4) << 3);
  ldsm_x4_t(r, base + row * ld + col);
}

// RG: a ragged batch (tq_attend_ragged).  A CTA takes one segment of the work
// list: its request's rows and lengths, key tiles [kt0, kt1) of one block of
// query positions; a tile cut into several segments leaves partial rows that
// the tile's last CTA joins.  Value norms enter P' times a power of two that puts
// the largest so far into [2^14, 2^15), and O keeps it through its last rotation:
// fp16 ends at 2^-24, where a cache's norms need not.
template <int D, int KB, int VB, bool RG, bool HP>
__global__ void __launch_bounds__(kPfThreads, 1) prefill_kernel(PrefillParams p) {
  using G = Pf<D, KB, VB, HP>;
  constexpr int NC = D / 16;                  // 16-wide chunks of D
  constexpr int NT = D / 8;                   // 8-wide n-tiles of D
  extern __shared__ __align__(128) unsigned char smem[];
  __half* Rs = reinterpret_cast<__half*>(smem + G::OFF_R);
  __half* Ks = reinterpret_cast<__half*>(smem + G::OFF_KS);
  __half* Vs = reinterpret_cast<__half*>(smem + G::OFF_VS);
  float* kn = reinterpret_cast<float*>(smem + G::OFF_NRM);
  float* vn = kn + 64;
  __half* lutk = reinterpret_cast<__half*>(smem + G::OFF_LUT);
  __half* lutv = lutk + 256;
  // HP: the low parts
  __half* Rl = reinterpret_cast<__half*>(smem + G::OFF_LO);
  __half* Kl = Rl + G::LO_K;
  __half* Vl = Rl + G::LO_V;
  __half* lutkl = Rl + G::LO_LUT;
  __half* lutvl = lutkl + 256;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::OFF_BAR);
  const uint32_t PAGE = (uint32_t)p.page_bytes;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  const int wph = kPfWarps / p.hc;                     // warps per head
  const int P = 16 * wph;                              // query positions per CTA
  const int nchunk = (int)(p.g / p.hc);
  SegWork sw = {};
  int qb = p.nqb - 1 - (int)blockIdx.x;                // long rows first
  int64_t group = blockIdx.y;                          // (b, kv head, chunk of its query heads)
  __shared__ int bad_key, last_flag;
  __shared__ int v_exp;                                // RG: value norms are scaled by 2^v_exp
  __shared__ float o_scale;                            // RG: what that changed by with this page
  if constexpr (RG) {
    if (!take_segment(p.rg, blockIdx.x, sw)) return;
    qb = sw.seg.tile;
    group = sw.seg.req * (p.Hkv * nchunk) + sw.group;
    p.Tq = sw.rq.q_len;
    p.n_tokens = sw.rq.seq;
    if (threadIdx.x == 0) {
      bad_key = INT_MAX;
      v_exp = 38;
    }
  }
  // rows and keys of the request: 32 bits hold a ragged batch's
  using Pos = typename std::conditional<RG, int, int64_t>::type;
  const int chunk = (int)(group % nchunk);
  const int64_t b = group / nchunk / p.Hkv, kvh = group / nchunk % p.Hkv;
  // stream of the keys (RG: the values' may differ, see fetch)
  const int64_t stream = RG ? b * p.rg.hv.streams + p.rg.hv.key_head((int)kvh) : group / nchunk;
  // the batch row's first query row: batch stride, or the request's first row
  const int64_t qrow = RG ? sw.rq.q0 * p.qs[2] : b * p.qs[0];
  const int64_t orow = RG ? sw.rq.q0 * p.os[2] : b * p.os[0];
  // head i of the CTA's, counted over all
  auto head = [&](int i) -> int64_t {
    return RG ? p.rg.hv.head((int)kvh, chunk * p.hc + i) : kvh * p.g + (int64_t)chunk * p.hc + i;
  };
  const int64_t h = head(warp / wph);                  // this warp's head
  const Pos t_base = RG ? (Pos)sw.rq.base : p.n_tokens - p.Tq;     // position of query 0
  const int t0 = qb * P + (warp % wph) * 16;           // this warp's first query
  const Pos qpos_max = t_base + tmin<Pos>((Pos)(qb + 1) * P, p.Tq) - 1;
  // keys this CTA needs
  const Pos kend = !p.causal ? p.n_tokens : RG ? tmin<Pos>(qpos_max + 1, p.n_tokens) : qpos_max + 1;
  const int tile0 = RG ? sw.seg.kt0 : 0;
  const int ntiles = RG ? sw.seg.kt1 - tile0 : (int)((kend + 63) / 64);
  Pos kst = 0;                                         // first attended key (left padding)
  if (p.kv_start) {
    const int v = __ldg(p.kv_start + b);
    kst = v < 0 ? 0 : v;
  }

  if (tid == 0) {
    mbar_init(&full[0], 1);
    mbar_init(&full[1], 1);
    fence_mbar_init();
  }
  // R (fp16) and the centroid tables
  if constexpr (HP) {
    for (int i = tid; i < D * D / 2; i += kPfThreads) {
      const int r = i / (D / 2), c = 2 * (i % (D / 2));
      const float* src = p.rot + r * D + c;
      uint32_t lo;
      *reinterpret_cast<uint32_t*>(Rs + r * G::LD + c) = split_half2(__ldg(src), __ldg(src + 1), lo);
      *reinterpret_cast<uint32_t*>(Rl + r * G::LD + c) = lo;
    }
  } else {
    for (int i = tid; i < D * D / 8; i += kPfThreads) {
      const int r = i / (D / 8), c8 = i % (D / 8);
      *reinterpret_cast<uint4*>(Rs + r * G::LD + c8 * 8) =
          __ldg(reinterpret_cast<const uint4*>(p.rot_h + r * D) + c8);
    }
  }
  for (int i = tid; i < 256; i += kPfThreads) {
    const float k = i < (1 << KB) ? __ldg(p.kc + i) : 0.f, v = i < (1 << VB) ? __ldg(p.vc + i) : 0.f;
    lutk[i] = __float2half_rn(k);
    lutv[i] = __float2half_rn(v);
    if constexpr (HP) {
      lutkl[i] = __float2half_rn(k - __half2float(lutk[i]));
      lutvl[i] = __float2half_rn(v - __half2float(lutv[i]));
    }
  }
  __syncthreads();
  // pool address of a stream's page pg (block table or contiguous)
  auto page_src = [&](int64_t of, int64_t pg) -> const uint8_t* {
    bool ok;
    const int64_t ps = page_slot(p.pm, of, pg + tile0, ok);
    if (!ok) atomicOr(p.status, TQ_DEV_BAD_BLOCK);
    return p.pages + ps * (int64_t)PAGE;
  };
  // page pg into stage i: whole, or its key and value parts from the two streams' pages
  auto fetch = [&](int i, int64_t pg) {
    unsigned char* dst = smem + G::OFF_STG + i * p.page_pitch;
    const uint8_t* src = page_src(stream, pg);
    const int64_t vstream = RG && p.rg.hv.own ? b * p.rg.hv.streams + p.rg.hv.value_head((int)kvh) : stream;
    if (vstream == stream) {
      mbar_expect_tx(&full[i], PAGE);
      bulk_g2s(dst, src, PAGE, &full[i]);
      return;
    }
    const uint8_t* vsrc = page_src(vstream, pg);
    constexpr uint32_t KS = 64 * G::KROW, VS = 64 * G::VROW, NS = 128;
    mbar_expect_tx(&full[i], KS + VS + 2 * NS);
    bulk_g2s(dst, src, KS, &full[i]);
    bulk_g2s(dst + p.off_kn, src + p.off_kn, NS, &full[i]);
    bulk_g2s(dst + p.off_v, vsrc + p.off_v, VS, &full[i]);
    bulk_g2s(dst + p.off_vn, vsrc + p.off_vn, NS, &full[i]);
  };
  if (tid == 0)
    for (int i = 0; i < 2 && i < ntiles; ++i) fetch(i, i);

  // ---- queries: q' = (scale q) R^T as fp16 A fragments (log2e folded in) ----
  const bool active = t0 < p.Tq;
  uint32_t qf[NC][4], ql[HP ? NC : 1][4];
  {
    const float sc = p.scale;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const int64_t qbase = qrow + (RG ? p.rg.hv.in_q((int)h) : h) * p.qs[1];
    const int r0 = t0 + gq, r1 = r0 + 8;
    auto ld2 = [&](int r, int c, uint32_t& lo) -> uint32_t {
      lo = 0u;
      if (r >= p.Tq) return 0u;
      const int64_t o = qbase + (int64_t)r * p.qs[2] + (int64_t)c * p.qs[3];
      const float x = sc * load_elem(p.q, p.q_dtype, o), y = sc * load_elem(p.q, p.q_dtype, o + p.qs[3]);
      if constexpr (HP) return split_half2(x, y, lo);
      return pack_half2(x, y);
    };
#pragma unroll
    for (int kc = 0; kc < NC; ++kc) {
      uint32_t a[4] = {0u, 0u, 0u, 0u}, al[4] = {0u, 0u, 0u, 0u};
      if (active) {
        a[0] = ld2(r0, 16 * kc + 2 * tq, al[0]);
        a[1] = ld2(r1, 16 * kc + 2 * tq, al[1]);
        a[2] = ld2(r0, 16 * kc + 2 * tq + 8, al[2]);
        a[3] = ld2(r1, 16 * kc + 2 * tq + 8, al[3]);
      }
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t bf[4];
        frag_b_nk(bf, Rs, G::LD, 8 * n, 16 * kc, lane);   // B[k][n] = R[n][k]
        mma_f16_16816(acc[n], a, bf[0], bf[1]);
        mma_f16_16816(acc[n + 1], a, bf[2], bf[3]);
        if constexpr (HP) {
          mma_f16_16816(acc[n], al, bf[0], bf[1]);
          mma_f16_16816(acc[n + 1], al, bf[2], bf[3]);
          frag_b_nk(bf, Rl, G::LD, 8 * n, 16 * kc, lane);
          mma_f16_16816(acc[n], a, bf[0], bf[1]);
          mma_f16_16816(acc[n + 1], a, bf[2], bf[3]);
        }
      }
    }
#pragma unroll
    for (int kc = 0; kc < NC; ++kc) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = acc[2 * kc + (i >> 1)][2 * (i & 1)] * kLog2eP;
        const float y = acc[2 * kc + (i >> 1)][2 * (i & 1) + 1] * kLog2eP;
        if constexpr (HP) qf[kc][i] = split_half2(x, y, ql[kc][i]);
        else qf[kc][i] = pack_half2(x, y);
      }
    }
  }

  float O[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) O[n][0] = O[n][1] = O[n][2] = O[n][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const Pos qp0 = t_base + t0 + gq, qp1 = qp0 + 8;               // query positions
  const Pos warp_kend = p.causal ? tmin<Pos>(t_base + t0 + 16, p.n_tokens) : p.n_tokens;

  int kt = 0;
  for (; kt < ntiles; ++kt) {
    const int st = kt & 1;
    // every thread observes the copy; the block agrees on a timeout
    const bool ok = mbar_wait_bounded(&full[st], (uint32_t)((kt >> 1) & 1));
    if (__syncthreads_or(!ok)) {
      if (tid == 0) atomicOr(p.status, TQ_DEV_WAIT_TIMEOUT);
      break;
    }
    const uint8_t* pg = smem + G::OFF_STG + st * p.page_pitch;
    // ---- decode K and V codes into fp16 tiles (coordinate order) ----------
    {
      // K: thread -> (token, quad); quad t of a row lists, for each chunk j,
      // coordinates 16j+2t, 16j+2t+1, 16j+2t+8, 16j+2t+9
      const int tok = tid >> 2, qd = tid & 3;
      constexpr int QB = (D / 4) * KB;                 // bits per quad
      const uint8_t* row = pg + tok * G::KROW;
      const int bit0 = qd * QB;
#pragma unroll
      for (int e = 0; e < D / 4; ++e) {
        const int bo = bit0 + e * KB;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(row + ((bo >> 5) << 2));
        uint32_t code;
        if ((bo & 31) + KB <= 32) {
          code = (w >> (bo & 31)) & ((1u << KB) - 1u);
        } else {
          const uint32_t w2 = *reinterpret_cast<const uint32_t*>(row + ((bo >> 5) << 2) + 4);
          code = __funnelshift_r(w, w2, bo & 31) & ((1u << KB) - 1u);
        }
        const int j = e >> 2, r = e & 3;
        const int coord = 16 * j + 2 * qd + (r & 1) + ((r >> 1) << 3);
        Ks[tok * G::LD + coord] = lutk[code];
        if constexpr (HP) Kl[tok * G::LD + coord] = lutkl[code];
      }
      // V: thread -> (token, two octets); octet o lists coordinates o, o+8, ...
      constexpr int OB = (D / 8) * VB;                 // bits per octet
      const uint8_t* vrow = pg + p.off_v + tok * G::VROW;
#pragma unroll
      for (int oo = 0; oo < 2; ++oo) {
        const int oct = 2 * qd + oo;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const int bo = oct * OB + c * VB;
          const uint32_t w = *reinterpret_cast<const uint32_t*>(vrow + ((bo >> 5) << 2));
          uint32_t code;
          if ((bo & 31) + VB <= 32) {
            code = (w >> (bo & 31)) & ((1u << VB) - 1u);
          } else {
            const uint32_t w2 = *reinterpret_cast<const uint32_t*>(vrow + ((bo >> 5) << 2) + 4);
            code = __funnelshift_r(w, w2, bo & 31) & ((1u << VB) - 1u);
          }
          Vs[tok * G::LD + oct + 8 * c] = lutv[code];
          if constexpr (HP) Vl[tok * G::LD + oct + 8 * c] = lutvl[code];
        }
      }
      if constexpr (RG) {
        // warp 0: value norms, warp 1: key norms, two tokens a lane
        if (warp < 2) {
          const __half* src = reinterpret_cast<const __half*>(pg + (warp == 0 ? p.off_vn : p.off_kn));
          float x[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int t = lane + 32 * i;
            const Pos key = (Pos)(kt + tile0) * 64 + t;
            x[i] = key < kend ? __half2float(src[t]) : 0.f;
            // 0 x inf would reach rows that do not see the key: a norm that is not
            // finite counts as 0 and the rows that see it become NaN at the end
            if (!isfinite(x[i])) {
              x[i] = 0.f;
              atomicMin(&bad_key, (int)key);
            }
          }
          if (warp == 0) {
            // the page's largest norm, below 2^(e + 1): the scale keeps it below 2^15
            const int e0 = v_exp;
            const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(x[0]), fabsf(x[1]))));
            const int e = tmin(e0, 14 - ((int)(top >> 23) - 127));
            const float scale = __uint_as_float((uint32_t)(127 + e) << 23);
            x[0] *= scale;
            x[1] *= scale;
            if (lane == 0) {
              o_scale = __uint_as_float((uint32_t)(127 + e - e0) << 23);
              v_exp = e;
            }
          }
          float* dst = warp == 0 ? vn : kn;
          dst[lane] = x[0];
          dst[lane + 32] = x[1];
        }
      } else if (tid < 64) {
        const int64_t key = (int64_t)(kt + tile0) * 64 + tid;
        const bool kok = key < kend;
        kn[tid] = kok ? __half2float(reinterpret_cast<const __half*>(pg + p.off_kn)[tid]) : 0.f;
        vn[tid] = kok ? __half2float(reinterpret_cast<const __half*>(pg + p.off_vn)[tid]) : 0.f;
      }
    }
    __syncthreads();
    // the stage is decoded: refill it with page kt + 2
    if (tid == 0 && kt + 2 < ntiles) fetch(st, kt + 2);

    const Pos k0 = (Pos)(kt + tile0) * 64;
    if constexpr (RG) {
      const float f = o_scale;                         // O follows the scale of the value norms
      if (f != 1.f) {
#pragma unroll
        for (int n = 0; n < NT; ++n) { O[n][0] *= f; O[n][1] *= f; O[n][2] *= f; O[n][3] *= f; }
      }
    }
    if (active && k0 < warp_kend) {
      // ---- S = Q' K^T (16 x 64) -------------------------------------------
      float s[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int kc = 0; kc < NC; ++kc) {
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
          uint32_t bf[4];
          frag_b_nk(bf, Ks, G::LD, 8 * n, 16 * kc, lane);
          mma_f16_16816(s[n], qf[kc], bf[0], bf[1]);
          mma_f16_16816(s[n + 1], qf[kc], bf[2], bf[3]);
          if constexpr (HP) {
            mma_f16_16816(s[n], ql[kc], bf[0], bf[1]);
            mma_f16_16816(s[n + 1], ql[kc], bf[2], bf[3]);
            frag_b_nk(bf, Kl, G::LD, 8 * n, 16 * kc, lane);
            mma_f16_16816(s[n], qf[kc], bf[0], bf[1]);
            mma_f16_16816(s[n + 1], qf[kc], bf[2], bf[3]);
          }
        }
      }
      // norms, causal mask, running max
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int kl = 8 * n + 2 * tq + c;
          const Pos key = k0 + kl;
          const float nk = kn[kl];
          float v0 = s[n][c] * nk, v1 = s[n][2 + c] * nk;
          const bool lim0 = key < p.n_tokens && key >= kst && (!p.causal || key <= qp0);
          const bool lim1 = key < p.n_tokens && key >= kst && (!p.causal || key <= qp1);
          v0 = lim0 ? v0 : -INFINITY;
          v1 = lim1 ? v1 : -INFINITY;
          s[n][c] = v0;
          s[n][2 + c] = v1;
          mx0 = fmaxf(mx0, v0);
          mx1 = fmaxf(mx1, v1);
        }
      }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      if (mx0 > m0) {
        const float c = fast_exp2(m0 - mx0);
        l0 *= c;
#pragma unroll
        for (int n = 0; n < NT; ++n) { O[n][0] *= c; O[n][1] *= c; }
        m0 = mx0;
      }
      if (mx1 > m1) {
        const float c = fast_exp2(m1 - mx1);
        l1 *= c;
#pragma unroll
        for (int n = 0; n < NT; ++n) { O[n][2] *= c; O[n][3] *= c; }
        m1 = mx1;
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      // ---- P' = P * ||v|| as A fragments; O += P' V ----------------------
      uint32_t pa[4][4], pl[HP ? 4 : 1][4];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int kl = 8 * n + 2 * tq;
        const float p00 = fast_exp2(s[n][0] - b0), p01 = fast_exp2(s[n][1] - b0);
        const float p10 = fast_exp2(s[n][2] - b1), p11 = fast_exp2(s[n][3] - b1);
        l0 += p00 + p01;
        l1 += p10 + p11;
        const float w0 = vn[kl], w1 = vn[kl + 1];
        const int i = (n & 1) * 2;
        if constexpr (HP) {
          pa[n >> 1][i] = split_half2(p00 * w0, p01 * w1, pl[n >> 1][i]);
          pa[n >> 1][i + 1] = split_half2(p10 * w0, p11 * w1, pl[n >> 1][i + 1]);
        } else {
          pa[n >> 1][i] = pack_half2(p00 * w0, p01 * w1);
          pa[n >> 1][i + 1] = pack_half2(p10 * w0, p11 * w1);
        }
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t a[4] = {pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3]};
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t bf[4];
          frag_b_kn(bf, Vs, G::LD, 8 * n, 16 * kk, lane);
          mma_f16_16816(O[n], a, bf[0], bf[1]);
          mma_f16_16816(O[n + 1], a, bf[2], bf[3]);
          if constexpr (HP) {
            mma_f16_16816(O[n], pl[kk], bf[0], bf[1]);
            mma_f16_16816(O[n + 1], pl[kk], bf[2], bf[3]);
            frag_b_kn(bf, Vl, G::LD, 8 * n, 16 * kk, lane);
            mma_f16_16816(O[n], a, bf[0], bf[1]);
            mma_f16_16816(O[n + 1], a, bf[2], bf[3]);
          }
        }
      }
    }
    __syncthreads();   // the tiles are rewritten by the next decode
  }
  // after a timeout, never leave with a copy still writing shared memory:
  // tiles kt and kt + 1 may still be in flight
  if (tid == 0 && kt < ntiles) {
    for (int i = kt; i < tmin(kt + 2, ntiles); ++i)
      mbar_wait_bounded(&full[i & 1], (uint32_t)((i >> 1) & 1), 16u);
  }

  // ---- O = (O' / l) R, stored -----------------------------------------------
  if (active) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    float i0 = l0 > 0.f ? 1.f / l0 : 0.f, i1 = l1 > 0.f ? 1.f / l1 : 0.f;
    if constexpr (RG) {
      const Pos last = p.n_tokens - 1;
      if (l0 != l0 || bad_key <= (p.causal ? tmin(qp0, last) : last)) l0 = i0 = NAN;
      if (l1 != l1 || bad_key <= (p.causal ? tmin(qp1, last) : last)) l1 = i1 = NAN;
    }
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
    for (int kc = 0; kc < NC; ++kc) {
      uint32_t a[4], al[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = O[2 * kc + (i >> 1)][2 * (i & 1)] * (i & 1 ? i1 : i0);
        const float y = O[2 * kc + (i >> 1)][2 * (i & 1) + 1] * (i & 1 ? i1 : i0);
        if constexpr (HP) a[i] = split_half2(x, y, al[i]);
        else a[i] = pack_half2(x, y);
      }
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t bf[4];
        frag_b_kn(bf, Rs, G::LD, 8 * n, 16 * kc, lane);   // B[k][n] = R[k][n]
        mma_f16_16816(acc[n], a, bf[0], bf[1]);
        mma_f16_16816(acc[n + 1], a, bf[2], bf[3]);
        if constexpr (HP) {
          mma_f16_16816(acc[n], al, bf[0], bf[1]);
          mma_f16_16816(acc[n + 1], al, bf[2], bf[3]);
          frag_b_kn(bf, Rl, G::LD, 8 * n, 16 * kc, lane);
          mma_f16_16816(acc[n], a, bf[0], bf[1]);
          mma_f16_16816(acc[n + 1], a, bf[2], bf[3]);
        }
      }
    }
    if constexpr (RG) {
      const float down = __uint_as_float((uint32_t)(127 - v_exp) << 23);
#pragma unroll
      for (int n = 0; n < NT; ++n) { acc[n][0] *= down; acc[n][1] *= down; acc[n][2] *= down; acc[n][3] *= down; }
    }
    const int r0 = t0 + gq, r1 = r0 + 8;
    const int64_t ocol = RG ? p.rg.hv.column((int)kvh, D) * p.os[3] : 0;
    const int64_t obase = orow + h * p.os[1] + ocol;
    const bool split = RG && sw.seg.slot >= 0;
    if (split) {
      const int64_t pr = part_row(p.rg.plan, sw.seg.slot, sw.group, 16 * warp + gq);
      float* part = p.rg.plan.part + pr * D + 2 * tq;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (r0 < p.Tq) *reinterpret_cast<float2*>(part + 8 * n) = make_float2(acc[n][0], acc[n][1]);
        if (r1 < p.Tq)
          *reinterpret_cast<float2*>(part + 8 * D + 8 * n) = make_float2(acc[n][2], acc[n][3]);
      }
      if (tq == 0) {
        if (r0 < p.Tq) p.rg.plan.ml[pr] = make_float2(m0, l0);
        if (r1 < p.Tq) p.rg.plan.ml[pr + 8] = make_float2(m1, l1);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (split) break;
      const int c = 8 * n + 2 * tq;
      if (r0 < p.Tq) {
        const int64_t o = obase + (int64_t)r0 * p.os[2] + (int64_t)c * p.os[3];
        store_elem(p.out, p.o_dtype, o, acc[n][0]);
        store_elem(p.out, p.o_dtype, o + p.os[3], acc[n][1]);
      }
      if (r1 < p.Tq) {
        const int64_t o = obase + (int64_t)r1 * p.os[2] + (int64_t)c * p.os[3];
        store_elem(p.out, p.o_dtype, o, acc[n][2]);
        store_elem(p.out, p.o_dtype, o + p.os[3], acc[n][3]);
      }
    }
  }
  if constexpr (RG) {
    if (sw.seg.slot >= 0)
      join_partials<D>(p.rg.plan, sw, kPfWarps, p.out, p.o_dtype, p.os[3], &last_flag,
                       [&](int row) -> int64_t {
                         const int wr = row >> 4, t = qb * P + (wr % wph) * 16 + (row & 15);
                         if (t >= p.Tq) return -1;
                         return orow + head(wr / wph) * p.os[1] + p.rg.hv.column((int)kvh, D) * p.os[3] +
                                t * p.os[2];
                       });
  }
}

using PfFn = void (*)(PrefillParams);

template <int D, bool RG, bool HP = false>
PfFn pf_fn(int kb, int vb) {
#define TQ_PF(K, V) if (kb == K && vb == V) return prefill_kernel<D, K, V, RG, HP>;
  TQ_PF(4, 2) TQ_PF(3, 3) TQ_PF(2, 2) TQ_PF(4, 4) TQ_PF(6, 4) TQ_PF(5, 5) TQ_PF(6, 6)
  TQ_PF(8, 8) TQ_PF(3, 2) TQ_PF(4, 3)
  // a ragged batch's fp16 and fp32 results have no tcgen05 kernel to take these
  if constexpr (RG) { TQ_PF(5, 4) }
#undef TQ_PF
  return nullptr;
}

}  // namespace

bool prefill_supported(int D, int kb, int vb) {
  if (D == 128) return pf_fn<128, false>(kb, vb) != nullptr;
  if (D == 64) return pf_fn<64, false>(kb, vb) != nullptr;
  return false;
}

bool attend_mma_applies(const tq_geom* G) {
  if (G->head_dim == 128) return pf_fn<128, true>(G->key_bits, G->value_bits) != nullptr;
  if (G->head_dim == 64) return pf_fn<64, true>(G->key_bits, G->value_bits) != nullptr;
  return false;
}

// Ragged batch on the mma.sync kernel; `grid` bounds the work list.  bf16 results
// take single fp16 operands (their rounding, 2^-12 of each, is a sixteenth of the
// result's own); fp16 and fp32 ones hi + lo.
int launch_attend_mma(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                      const tq_attend_args* a, bool precise, const RaggedAttend& rg, int64_t Hkv,
                      int hc, int64_t grid, uint32_t* status, cudaStream_t st) {
  PrefillParams p = {};
  const PageGeom g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.pages = c->pages;
  p.pm = page_map(c);
  p.page_bytes = g.page_bytes;
  p.page_pitch = (g.page_bytes + 127) & ~127;
  p.off_v = g.off_v;
  p.off_kn = g.off_kn;
  p.off_vn = g.off_vn;
  p.rot_h = reinterpret_cast<const __half*>(t->rot_f16);
  p.kc = t->k_centroids;
  p.vc = t->v_centroids;
  p.q = a->q->data; p.q_dtype = a->q->dtype;
  p.out = a->out->data; p.o_dtype = a->out->dtype;
  for (int i = 0; i < 4; ++i) { p.qs[i] = a->q->stride[i]; p.os[i] = a->out->stride[i]; }
  p.Hq = a->q->shape[1];
  p.Hkv = Hkv;
  p.g = rg.hv.g;
  p.hc = hc;
  p.scale = a->scale;
  p.causal = a->causal;
  p.status = status;
  p.rg = rg;
  p.rot = t->rot;
  const int kb = G->key_bits, vb = G->value_bits;
  const bool wide = G->head_dim == 128;
  PfFn fn;
  int smem;
  if (precise) {
    fn = wide ? pf_fn<128, true, true>(kb, vb) : pf_fn<64, true, true>(kb, vb);
    smem = wide ? Pf<128, 4, 4, true>::smem(p.page_pitch) : Pf<64, 4, 4, true>::smem(p.page_pitch);
  } else {
    fn = wide ? pf_fn<128, true>(kb, vb) : pf_fn<64, true>(kb, vb);
    smem = wide ? Pf<128, 4, 4, false>::smem(p.page_pitch) : Pf<64, 4, 4, false>::smem(p.page_pitch);
  }
  if (set_smem_attr((const void*)fn, smem) != TQ_OK) return TQ_ERR_CUDA;
  fn<<<(unsigned)grid, kPfThreads, smem, st>>>(p);
  return check_launch("tq_attend_ragged");
}

int launch_prefill(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                   const tq_prefill_args* a, uint32_t* status, cudaStream_t st) {
  if (a->engine != 1) {
    const int rc = launch_prefill_tc(G, t, c, a, status, st);
    if (rc != 1) return rc;
  }
  PrefillParams p = {};
  const PageGeom g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.pages = c->pages;
  p.pm = page_map(c);
  p.page_bytes = g.page_bytes;
  p.page_pitch = (g.page_bytes + 127) & ~127;
  p.off_v = g.off_v;
  p.off_kn = g.off_kn;
  p.off_vn = g.off_vn;
  p.rot_h = reinterpret_cast<const __half*>(t->rot_f16);
  p.kc = t->k_centroids;
  p.vc = t->v_centroids;
  p.q = a->q->data; p.q_dtype = a->q->dtype;
  p.out = a->out->data; p.o_dtype = a->out->dtype;
  for (int i = 0; i < 4; ++i) { p.qs[i] = a->q->stride[i]; p.os[i] = a->out->stride[i]; }
  p.Hq = a->q->shape[1];
  p.Hkv = c->streams / a->q->shape[0];
  p.g = a->q->shape[1] / p.Hkv;
  p.hc = p.g % 8 == 0 ? 8 : p.g % 4 == 0 ? 4 : p.g % 2 == 0 ? 2 : 1;
  p.Tq = a->q->shape[2];
  p.n_tokens = a->n_tokens;
  p.scale = a->scale;
  p.causal = a->causal;
  p.kv_start = a->kv_start;
  p.nqb = (int)((p.Tq + 16 * (kPfWarps / p.hc) - 1) / (16 * (kPfWarps / p.hc)));
  p.status = status;
  if (p.Tq == 0) return TQ_OK;
  PfFn fn = G->head_dim == 128 ? pf_fn<128, false>(G->key_bits, G->value_bits)
                               : pf_fn<64, false>(G->key_bits, G->value_bits);
  const int smem = G->head_dim == 128 ? Pf<128, 4, 4, false>::smem(p.page_pitch)
                                      : Pf<64, 4, 4, false>::smem(p.page_pitch);
  if (!fn) {
    set_error("tq_prefill_attn: no kernel for head_dim %d, key_bits %d, value_bits %d",
              G->head_dim, G->key_bits, G->value_bits);
    return TQ_ERR_INVALID;
  }
  if (set_smem_attr((const void*)fn, smem) != TQ_OK) return TQ_ERR_CUDA;
  dim3 grid((unsigned)p.nqb, (unsigned)(a->q->shape[0] * p.Hq / p.hc));
  fn<<<grid, kPfThreads, smem, st>>>(p);
  return check_launch("tq_prefill_attn");
}

}  // namespace tq
