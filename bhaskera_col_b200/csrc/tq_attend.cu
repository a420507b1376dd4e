// tq_attend.cu — attention of a ragged batch over the packed pages
// (tq_attend_ragged): the work list, its workspace and the choice of kernel.
//
// A tile is one request's block of `pcta` query positions with the query heads
// of one head group; it attends ceil(keys / kt) key tiles.  With few rows and
// long contexts there are far fewer tiles than SMs, so tiles are cut along the
// keys into segments of at most L key tiles,
//     L = max(kMinTiles, ceil(all key tiles / wanted CTAs)),
// one CTA each.  The list is built on the device (the lengths live there), so
// the host neither waits nor reads them; it launches an upper bound of CTAs.
// Two kernels may share a batch: requests of few query rows take tiles of 8 or 16
// rows (tq_attend_few.cu), the others tiles of 256 (tcgen05), each from a list of
// its own.
#include "tq_internal.h"
#include "tq_ragged.cuh"

#include <initializer_list>

namespace tq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr unsigned long long kOneTile = 1ull << 40;   // tiles counted above their key tiles
constexpr int kClasses = 32;               // length classes of segments
// Segments wanted per SM (more even the ends, fewer save set-ups and joins) and the
// shortest segment worth a CTA's set-up, in keys.  Wide list, 8,899 rows of prompt
// chunks: 605 us with 2 a SM, 611 with 1, 660 with 3, 720 with 5.  Few-row list
// (three CTAs a SM): 131,001 keys 142 us with 5 a SM, 172 with 3, 157 with 8; 64
// requests' drafts 163, 166, 168.  Shortest: one request of 2,000 keys 35 us with 512,
// 33 with 256, 43 with 1,024; 64 of 1,000 keys 46, 57, 47.
// Other batches, wide list with 1, 2, 3, 5 a SM: one prompt of 8,100 rows 934, 927,
// 924, 1,039 us; four of 2,000 over 4,000 keys each 1,219, 1,228, 1,225, 1,225; forty of
// 300 595, 595, 595, 650.  Few-row list with 3, 5, 8: one token over 32,771 keys 35, 45,
// 46; 8 x 4 over 15,999 87, 77, 85; 32 over up to 9,000 58, 53, 60; 256 over up to
// 2,000 60, 61, 61; 64 over 8,000 183, 163, 161; full attention of 100 x 20 rows, heads
// of 64, 76, 76, 84.
constexpr int kWaves = 2, kMinKeys = 512;
constexpr int kFewWaves = 5, kFewMinKeys = 512;

struct PlanParams {
  RaggedView rv;
  int64_t q_lo, q_hi;                      // the list's requests: q_lo < q_len <= q_hi
  int pcta, keys, key_shift;               // query positions per tile, keys per key tile (2^shift)
  int causal, G;
  int64_t wanted;                          // segments wanted, all head groups together
  int min_tiles, max_seg, max_slot;
  RaggedSeg* segs;
  int32_t* nseg;
  int32_t* next;
  int32_t* arrived;
  uint32_t* status;
};

// A listed request in the plan's terms.
struct Tiles {
  int tiles, q_len, seq, base;
};

__device__ __forceinline__ Tiles listed_request(const PlanParams& p, int64_t r) {
  Tiles t = {0, 0, 0, 0};
  if (r >= p.rv.R) return t;
  const Request q = request_at(p.rv, r);
  if (q.q_len <= p.q_lo || q.q_len > p.q_hi) return t;
  t.q_len = (int)q.q_len;
  t.seq = (int)q.seq;
  t.base = (int)q.base;
  if (t.base + t.q_len > t.seq) atomicOr(p.status, TQ_DEV_BAD_POSITION);   // longer than its pages
  t.tiles = (t.q_len + p.pcta - 1) / p.pcta;
  return t;
}

// Key tiles of query block i.
__device__ __forceinline__ int key_tiles(const PlanParams& p, const Tiles& t, int i) {
  int kend = t.seq;
  if (p.causal) kend = tmin(kend, t.base + (int)tmin<int64_t>((int64_t)(i + 1) * p.pcta, t.q_len));
  return kend > 0 ? (kend + p.keys - 1) >> p.key_shift : 0;
}

// f(request, tile, key tiles) for every tile: a thread per request, a warp
// for a request of more than 32 tiles.  `own`: this thread's first request, read
// once for all passes.
template <class F>
__device__ __forceinline__ void for_tiles(const PlanParams& p, const Tiles& own, F f) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int64_t r0 = 0; r0 < p.rv.R; r0 += kPlanThreads) {
    const Tiles t = r0 == 0 ? own : listed_request(p, r0 + tid);
    if (t.tiles <= 32)
      for (int i = 0; i < t.tiles; ++i) f((int)(r0 + tid), i, key_tiles(p, t, i));
    for (unsigned big = __ballot_sync(0xffffffffu, t.tiles > 32); big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Tiles b;
      b.tiles = __shfl_sync(0xffffffffu, t.tiles, src);
      b.q_len = __shfl_sync(0xffffffffu, t.q_len, src);
      b.seq = __shfl_sync(0xffffffffu, t.seq, src);
      b.base = __shfl_sync(0xffffffffu, t.base, src);
      for (int i = lane; i < b.tiles; i += 32) f((int)(r0 + (tid & ~31) + src), i, key_tiles(p, b, i));
    }
  }
}

// ---------------------------------------------------------------------------
// q' = scale log2(e) q R^T of the few-row list's queries, fp16 in quad order:
// CTAs of the plan's launch beside the lists' own.
// ---------------------------------------------------------------------------
struct QueryParams {
  const void* q; int q_dtype; int q_vec; int64_t qs[3];    // head, row, dim; 16-byte pieces
  const __half* rot_h;
  const float* rot;                                        // for hi + lo, or NULL
  __half* qp;                                              // [token][Hq][D], or [2][D] of hi and lo
  int64_t qp_stride;                                       // FewParams::qp_stride
  float qscale;
  int Hq, D, blocks;                                       // blocks of 64 rows looked at per request
};

constexpr int kQRows = 64;

__device__ __forceinline__ uint32_t split_half2(float a, float b, uint32_t& lo) {
  const uint32_t hi = pack_half2(a, b);
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  lo = pack_half2(a - __low2float(h), b - __high2float(h));
  return hi;
}

// 32 warps: four tiles of 16 rows, eight warps each, every eighth 8-wide slice
// of the result.  HP: q and R as fp16 hi + lo (three products), so is q'.
template <int D, bool HP>
__device__ __forceinline__ void rotate_queries(const PlanParams& p, const QueryParams& qp, int first,
                                               int step, unsigned char* sm) {
  constexpr int LD = D + 8;                                // halves per staged row (banks)
  __half* A = reinterpret_cast<__half*>(sm);
  __half* Al = A + kQRows * LD;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  for (int64_t item = first; item < p.rv.R * qp.blocks; item += step) {
    const int64_t r = item / qp.blocks;
    const Request rq = request_at(p.rv, r);
    if (rq.q_len <= p.q_lo || rq.q_len > p.q_hi) continue;
    const int64_t tok0 = qp.qp_stride ? r * qp.qp_stride : rq.q0;
    const int64_t rows = rq.q_len * qp.Hq;
    for (int64_t row0 = (item % qp.blocks) * kQRows; row0 < rows; row0 += (int64_t)qp.blocks * kQRows) {
      __syncthreads();
      for (int i = tid; i < kQRows * D / 8; i += kPlanThreads) {
        const int n = i / (D / 8), c = i % (D / 8);
        const int row = (int)row0 + n;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row < rows) {
          const int tok = row / qp.Hq, h = row - tok * qp.Hq;
          const int64_t at = (rq.q0 + tok) * qp.qs[1] + h * qp.qs[0] + (int64_t)(8 * c) * qp.qs[2];
          if (qp.q_vec) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(qp.q) + at));
            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 y = qp.q_dtype == TQ_F16
                                   ? __half22float2(*reinterpret_cast<const __half2*>(&u[e]))
                                   : make_float2(__uint_as_float(u[e] << 16),
                                                 __uint_as_float(u[e] & 0xFFFF0000u));
              f[2 * e] = y.x;
              f[2 * e + 1] = y.y;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = load_elem(qp.q, qp.q_dtype, at + e * qp.qs[2]);
          }
        }
        uint32_t w[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = split_half2(f[2 * e] * qp.qscale, f[2 * e + 1] * qp.qscale, l[e]);
        *reinterpret_cast<uint4*>(A + n * LD + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (HP) *reinterpret_cast<uint4*>(Al + n * LD + 8 * c) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      __syncthreads();
      const int m0 = 16 * (warp >> 3);
      for (int jt = warp & 7; jt < D / 8; jt += 8) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t b[D / 16][2];
        auto frag = [&](uint32_t (&a)[4], const __half* at, int ch) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[i] = *reinterpret_cast<const uint32_t*>(at + (m0 + gq + 8 * (i & 1)) * LD + 16 * ch +
                                                      2 * tq + 8 * (i >> 1));
        };
        uint32_t a[4];
        if constexpr (HP) {
          const float2* R = reinterpret_cast<const float2*>(qp.rot + (8 * jt + gq) * D) + tq;
          uint32_t bl[D / 16][2];
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 x = __ldg(R + 8 * ch + 4 * i);
              b[ch][i] = split_half2(x.x, x.y, bl[ch][i]);
            }
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch) {
            frag(a, A, ch);
            mma_f16_16816(c, a, b[ch][0], b[ch][1]);
            mma_f16_16816(c, a, bl[ch][0], bl[ch][1]);
            frag(a, Al, ch);
            mma_f16_16816(c, a, b[ch][0], b[ch][1]);
          }
        } else {
          const uint32_t* R = reinterpret_cast<const uint32_t*>(qp.rot_h + (8 * jt + gq) * D) + tq;
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch) {
            b[ch][0] = __ldg(R + 8 * ch);
            b[ch][1] = __ldg(R + 8 * ch + 4);
          }
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch) {
            frag(a, A, ch);
            mma_f16_16816(c, a, b[ch][0], b[ch][1]);
          }
        }
        // dims 8 jt + 2 tq, + 1: word jt of quad tq
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t row = row0 + m0 + gq + 8 * i;
          if (row < rows) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(qp.qp + (tok0 * qp.Hq + row) * (HP ? 2 * D : D)) +
                            tq * (D / 8) + jt;
            uint32_t lo;
            dst[0] = split_half2(c[2 * i], c[2 * i + 1], lo);
            if constexpr (HP) dst[D / 2] = lo;
          }
        }
      }
    }
  }
}

// One CTA per list (and the queries' CTAs).  Pass 0 sums the key tiles, pass 1 counts the segments of
// each length class, pass 2 writes them, long classes first (whatever is taken
// last should be short).  Places within a class come from atomics, so the
// order varies from run to run; results do not depend on it: a tile's segments
// have consecutive slots and are joined in slot order.
__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(PlanParams p0, PlanParams p1,
                                                                   int lists, QueryParams qp) {
  pdl_launch_dependents();
  if ((int)blockIdx.x >= lists) {
    __shared__ __align__(16) unsigned char sm[2 * kQRows * (128 + 8) * 2];
    const int first = blockIdx.x - lists, step = gridDim.x - lists;
    if (qp.D == 128 && qp.rot) rotate_queries<128, true>(p0, qp, first, step, sm);
    else if (qp.D == 128) rotate_queries<128, false>(p0, qp, first, step, sm);
    else if (qp.rot) rotate_queries<64, true>(p0, qp, first, step, sm);
    else rotate_queries<64, false>(p0, qp, first, step, sm);
    return;
  }
  const PlanParams& p = blockIdx.x == 0 ? p0 : p1;
  __shared__ unsigned long long all;
  __shared__ unsigned place[kClasses + 1];                 // segments per class, then their next place
  __shared__ unsigned slots;
  const int tid = threadIdx.x, lane = tid & 31;
  const OffsetCheck offsets(p.rv, tid);
  const Tiles own = listed_request(p, tid);
  for (int i = tid; i < p.max_slot * p.G; i += kPlanThreads) p.arrived[i] = 0;
  if (tid == 0) {
    all = 0;
    slots = 0;
    *p.next = 0;
  }
  if (tid <= kClasses) place[tid] = 0;
  if (__syncthreads_or(offsets.fails(p.rv, tid, kPlanThreads, p.status))) {
    if (tid == 0) *p.nseg = 0;
    return;
  }
  unsigned long long mine = 0;
  for_tiles(p, own, [&](int, int, int nkt) { mine += nkt + kOneTile; });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) atomicAdd(&all, mine);
  __syncthreads();
  const unsigned long long total = (all & (kOneTile - 1)) * (unsigned)p.G;
  // tiles that fill half of the wanted CTAs by themselves need no short segments
  // (16 batches of encoder states, 304 rows: 36.7 us, with them 41.2)
  const int least = (all / kOneTile) * (unsigned)p.G * 2 >= p.wanted ? 2 * p.min_tiles : p.min_tiles;
  const int L = (int)tmax<unsigned long long>(least, (total + p.wanted - 1) / p.wanted);
  // class of a segment of n key tiles: 0 the longest (L), 31 the shortest
  auto class_of = [&](int n) { return kClasses - 1 - (int)((unsigned)(n * kClasses - 1) / (unsigned)L); };
  for_tiles(p, own, [&](int, int, int nkt) {
    const int ns = nkt > L ? (nkt + L - 1) / L : 1;
    atomicAdd(&place[class_of(tmax(1, (nkt + ns - 1) / ns))], (unsigned)ns);
    if (ns > 1) atomicAdd(&slots, (unsigned)ns);
  });
  __syncthreads();
  if (tid < 32) {
    // exclusive sums of the classes; the bounds of the list hold for offsets that
    // ascend and stay as they were read
    const unsigned own = place[lane];
    unsigned x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    place[lane] = x - own;
    if (lane == 31) {
      const bool ok = x <= (unsigned)p.max_seg && slots <= (unsigned)p.max_slot;
      if (!ok) atomicOr(p.status, TQ_DEV_BAD_BATCH);
      place[kClasses] = ok;
      *p.nseg = ok ? (int)x : 0;
      slots = 0;
    }
  }
  __syncthreads();
  if (!place[kClasses]) return;
  for_tiles(p, own, [&](int r, int i, int nkt) {
    const int ns = nkt > L ? (nkt + L - 1) / L : 1;
    const int base = nkt / ns, more = nkt - base * ns;     // `more` segments take one tile extra
    const unsigned at = atomicAdd(&place[class_of(tmax(1, (nkt + ns - 1) / ns))], (unsigned)ns);
    const unsigned slot = ns > 1 ? atomicAdd(&slots, (unsigned)ns) : 0;
    int kt = 0;
    for (int s = 0; s < ns; ++s) {
      RaggedSeg g;
      g.req = r;
      g.tile = i;
      g.kt0 = kt;
      kt += base + (s < more);
      g.kt1 = kt;
      g.slot = ns > 1 ? (int)slot + s : -1;
      g.first = (int)slot;
      g.parts = ns;
      g.pad = 0;
      p.segs[at + s] = g;
    }
  });
}

// Shape of one list's launch: head group, query positions and rows of a CTA,
// the bounds of the work list and its place in the workspace.
struct ListShape {
  bool used;
  int64_t q_lo, q_hi;
  int hc, pcta, rows, keys, G;
  int64_t wanted, max_seg, max_slot;
  size_t off_nseg, off_segs, off_arrived, off_ml, off_part, off_qp;
};

struct AttendShape {
  bool tc;                                 // the wide list runs on tcgen05
  int64_t Hkv, qp_stride;
  ListShape few, wide;
  size_t bytes;
};

// Query rows of a request and KV head up to which the few-row kernel is taken
// where the tcgen05 kernel could be: 16 requests of 3,000-5,000 keys, D128, four
// heads a group: 64 rows 128 us against 197, 128 rows 199 against 227, 256 rows 375
// against 282.  Elsewhere it takes every request: the mma.sync kernel, which it
// replaces there, is behind at any number of rows (D64: 16 rows 41 us against 233,
// 1,024 rows 927 against 1,427; D128, fp16 results, 1,024 rows 3,281 against 3,925)
// and runs the codes that the few-row kernel has no table for (above 4 bits).
constexpr int kFewRows = 128;

// The kernels that a call may use: few rows, and tcgen05 (else mma.sync) for the
// others.  The tcgen05 kernel's operands are single fp16 values: for fp16 and fp32
// results (error 7e-4, against 2.1e-4 of fp16's own rounding) only when asked for,
// although it is six times as fast from 1,024 rows on (549 us against 3,281).
struct Kernels {
  bool few, tc;
};

Kernels attend_kernels(const tq_geom* G, const tq_attend_args* a) {
  Kernels k;
  k.few = attend_few_applies(G) && (a->engine == 0 || a->engine == 3);
  k.tc = prefill_tc_applies(G) && (a->engine == 2 || (a->engine == 0 && !attend_precise(a)));
  return k;
}

AttendShape attend_shape(const tq_geom* G, const tq_cache* c, const tq_attend_args* a) {
  AttendShape s = {};
  const int64_t R = a->batch.requests, N = a->q->shape[2], most = INT64_MAX;
  s.Hkv = c->streams / R;
  const int64_t g = a->q->shape[1] / s.Hkv;
  const Kernels kernels = attend_kernels(G, a);
  s.tc = kernels.tc;
  const bool can = kernels.few;
  const int64_t few_q = s.tc ? tmax<int64_t>(kFewRows / g, 1) : most;
  size_t off = 256;                        // the first 64 bytes: the decode's status word
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) & ~(size_t)255;
    return at;
  };
  auto finish = [&](ListShape& l) {
    l.used = true;
    l.G = (int)(s.Hkv * ((g + l.hc - 1) / l.hc));
    // tiles: one per started block of positions; L cuts off at most wanted / G
    // segments beyond them, and a cut tile has at most twice its extra ones
    const int64_t extra = l.wanted / l.G + 1;
    l.max_seg = N / l.pcta + R + extra;
    l.max_slot = 2 * extra;
    l.off_segs = take(l.max_seg * sizeof(RaggedSeg));
    l.off_arrived = take(l.max_slot * l.G * 4);
    l.off_ml = take((size_t)l.max_slot * l.G * l.rows * 8);
    l.off_part = take((size_t)l.max_slot * l.G * l.rows * G->head_dim * 4);
  };
  const bool wide = !can || a->batch.max_q_len > few_q;
  if (can) {
    ListShape& l = s.few;
    l.q_hi = wide ? few_q : most;
    l.rows = g * a->batch.max_q_len <= 8 ? 8 : 16;
    l.hc = (int)tmin<int64_t>(g, l.rows);
    l.pcta = l.rows / l.hc;
    l.keys = kPageTokens;
    l.wanted = (int64_t)kFewWaves * device_sm_count();
    l.off_nseg = 64;
    finish(l);
    // q' rows of its tokens: beside a wide list at most few_q of each request
    s.qp_stride = wide ? few_q : 0;
    l.off_qp = take((size_t)(wide ? R * few_q : N) * a->q->shape[1] * G->head_dim *
                    (attend_precise(a) ? 4 : 2));
  }
  if (wide) {
    ListShape& l = s.wide;
    l.q_lo = can ? few_q : 0;
    l.q_hi = most;
    // both kernels take 8, 4, 2 or 1 heads; the tcgen05 one two tiles of 128
    // rows that share their keys
    l.hc = g % 8 == 0 ? 8 : g % 4 == 0 ? 4 : g % 2 == 0 ? 2 : 1;
    l.rows = s.tc ? 256 : 128;
    l.pcta = l.rows / l.hc;
    l.keys = s.tc ? 2 * kPageTokens : kPageTokens;
    l.wanted = (int64_t)kWaves * device_sm_count();
    l.off_nseg = 72;
    finish(l);
  }
  s.bytes = off;
  return s;
}

}  // namespace

bool attend_applies(const tq_geom* G, const tq_attend_args* a) {
  const Kernels k = attend_kernels(G, a);
  return k.few || k.tc || (a->engine <= 1 && attend_mma_applies(G));
}

size_t attend_ragged_workspace(const tq_geom* G, const tq_cache* c, const tq_attend_args* a) {
  return attend_shape(G, c, a).bytes;
}

int launch_attend_ragged(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                         const tq_attend_args* a, void* ws, uint32_t* status, cudaStream_t st) {
  const AttendShape s = attend_shape(G, c, a);
  if (a->q->shape[2] == 0) return TQ_OK;
  uint8_t* base = static_cast<uint8_t*>(ws);
  RaggedAttend rg[2];
  PlanParams plan[2];
  int lists = 0;
  for (const ListShape* l : {&s.few, &s.wide}) {
    if (!l->used) continue;
    PlanParams& p = plan[lists];
    p.rv = ragged_view(&a->batch, a->q->shape[2], c);
    p.q_lo = l->q_lo;
    p.q_hi = l->q_hi;
    p.pcta = l->pcta;
    p.keys = l->keys;
    p.causal = a->causal;
    p.G = l->G;
    p.wanted = l->wanted;
    p.min_tiles = (l == &s.few ? kFewMinKeys : kMinKeys) / l->keys;
    p.max_seg = (int)l->max_seg;
    p.max_slot = (int)l->max_slot;
    p.nseg = reinterpret_cast<int32_t*>(base + l->off_nseg);
    p.next = p.nseg + 1;
    p.key_shift = l->keys == 64 ? 6 : 7;
    p.segs = reinterpret_cast<RaggedSeg*>(base + l->off_segs);
    p.arrived = reinterpret_cast<int32_t*>(base + l->off_arrived);
    p.status = status;
    RaggedAttend& r = rg[lists++];
    r.rv = p.rv;
    r.plan.segs = p.segs;
    r.plan.nseg = p.nseg;
    r.plan.next = p.next;
    r.plan.arrived = p.arrived;
    r.plan.ml = reinterpret_cast<float2*>(base + l->off_ml);
    r.plan.part = reinterpret_cast<float*>(base + l->off_part);
    r.plan.G = l->G;
    r.plan.rows = l->rows;
  }
  QueryParams qp = {};
  int query_ctas = 0;
  if (s.few.used) {
    qp.q = a->q->data;
    qp.q_dtype = a->q->dtype;
    for (int i = 0; i < 3; ++i) qp.qs[i] = a->q->stride[i + 1];
    qp.q_vec = qp.q_dtype != TQ_F32 && qp.qs[2] == 1 && reinterpret_cast<uintptr_t>(qp.q) % 16 == 0 &&
               qp.qs[0] % 8 == 0 && qp.qs[1] % 8 == 0;
    qp.rot_h = reinterpret_cast<const __half*>(t->rot_f16);
    qp.rot = attend_precise(a) ? t->rot : nullptr;
    qp.qp = reinterpret_cast<__half*>(base + s.few.off_qp);
    qp.qp_stride = s.qp_stride;
    qp.qscale = a->scale * 1.4426950408889634f;
    qp.Hq = (int)a->q->shape[1];
    qp.D = G->head_dim;
    const int64_t most = s.qp_stride ? s.qp_stride : tmax<int64_t>(a->batch.max_q_len, 1);
    qp.blocks = (int)tmin<int64_t>((most * qp.Hq + kQRows - 1) / kQRows, 1 << 16);
    query_ctas = (int)tmin<int64_t>(a->batch.requests * qp.blocks, device_sm_count());
  }
  ragged_plan_kernel<<<lists + query_ctas, kPlanThreads, 0, st>>>(plan[0], plan[lists - 1], lists, qp);
  if (check_launch("tq_attend_ragged/plan") != TQ_OK) return TQ_ERR_CUDA;
  if (s.few.used) {
    const int rc = launch_attend_few(G, t, c, a, rg[0], s.Hkv, s.few.hc, s.few.pcta, s.few.rows,
                                     qp.qp, s.qp_stride, s.few.max_seg * s.few.G, status, st);
    if (rc != TQ_OK) return rc;
  }
  if (s.wide.used && s.tc)
    return launch_attend_tc(G, t, c, a, rg[lists - 1], s.Hkv, s.wide.max_seg * s.wide.G, status,
                            st);
  if (s.wide.used)
    return launch_attend_mma(G, t, c, a, rg[lists - 1], s.Hkv, s.wide.hc,
                             s.wide.max_seg * s.wide.G, status, st);
  return TQ_OK;
}

}  // namespace tq
