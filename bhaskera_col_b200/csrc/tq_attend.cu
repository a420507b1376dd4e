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
// Two kernels share a batch: requests of few query rows take tiles of 8 or 16
// rows (tq_attend_few.cu), the others tiles of 128 or more, each from a list of
// its own.
#include "tq_internal.h"
#include "tq_ragged.cuh"

#include <initializer_list>

namespace tq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kWaves = 3;                  // segments wanted per SM
constexpr int kMinKeys = 512;              // shortest segment worth a CTA's set-up
constexpr int kFewWaves = 6, kFewMinKeys = 512;   // the same for the few-row kernel

struct PlanParams {
  RaggedView rv;
  int64_t q_lo, q_hi;                      // the list's requests: q_lo < q_len <= q_hi
  int pcta, keys;                          // query positions per tile, keys per key tile
  int causal, G;
  int64_t wanted;                          // segments wanted, all head groups together
  int min_tiles, max_seg, max_slot;
  RaggedSeg* segs;
  int32_t* nseg;
  int32_t* arrived;
  uint32_t* status;
};

// Key tiles of query block i of a request.
__device__ __forceinline__ int key_tiles(const PlanParams& p, const Request& q, int64_t i) {
  int64_t kend = q.seq;
  if (p.causal) kend = q.seq - q.q_len + tmin<int64_t>((i + 1) * p.pcta, q.q_len);
  return kend > 0 ? (int)((kend + p.keys - 1) / p.keys) : 0;
}

// Request r, empty where it belongs to the other list.
__device__ __forceinline__ Request listed_request(const PlanParams& p, int64_t r) {
  Request q = {};
  if (r < p.rv.R) q = request_at(p.rv, r);
  if (q.q_len <= p.q_lo || q.q_len > p.q_hi) q.q_len = 0;
  return q;
}

// Inclusive scan over the block of a pair of counts packed as hi:lo 32 bits.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* warp_tot, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_tot[warp] = x;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += warp_tot[w];
    total += warp_tot[w];
  }
  __syncthreads();
  return x + before;
}

// One CTA, one thread per request; a request of more than 32 tiles is walked
// by its whole warp.  Pass 0 sums the key tiles, pass 1 counts and writes the
// segments (in request and tile order: the list does not depend on timing).
__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(PlanParams p0, PlanParams p1) {
  const PlanParams& p = blockIdx.x == 0 ? p0 : p1;         // one CTA per list
  __shared__ uint64_t warp_tot[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < p.max_slot * p.G; i += kPlanThreads) p.arrived[i] = 0;
  // f(request, tile, lane's turn) for every tile of this thread's request
  uint64_t total = 0, sum = 0;
  for (int64_t r0 = 0; r0 < p.rv.R; r0 += kPlanThreads) {
    const int64_t r = r0 + tid;
    const Request q = listed_request(p, r);
    const int64_t tiles = (q.q_len + p.pcta - 1) / p.pcta;
    uint64_t mine = 0;
    if (tiles <= 32)
      for (int64_t i = 0; i < tiles; ++i) mine += key_tiles(p, q, i);
    for (unsigned big = __ballot_sync(0xffffffffu, tiles > 32); big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Request bq;
      bq.q0 = 0;
      bq.q_len = __shfl_sync(0xffffffffu, q.q_len, src);
      bq.seq = __shfl_sync(0xffffffffu, q.seq, src);
      const int64_t bt = __shfl_sync(0xffffffffu, tiles, src);
      uint64_t part = 0;
      for (int64_t i = lane; i < bt; i += 32) part += key_tiles(p, bq, i);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == src) mine = part;
    }
    block_scan(mine, warp_tot, sum);
    total += sum;
  }
  const int64_t all = (int64_t)total * p.G;
  const int L = (int)tmax<int64_t>(p.min_tiles, (all + p.wanted - 1) / p.wanted);

  // segments (low word) and partial slots (high word) of one tile
  auto cuts = [&](int nkt) -> uint64_t {
    const uint64_t ns = nkt > L ? (uint64_t)((nkt + L - 1) / L) : 1;
    return ns | (ns > 1 ? ns << 32 : 0);
  };
  auto put = [&](int64_t r, int64_t i, int nkt, uint64_t at) {
    const int ns = (int)(uint32_t)cuts(nkt);
    const int64_t seg = (uint32_t)at, slot = (uint32_t)(at >> 32);
    if (seg + ns > p.max_seg || (ns > 1 && slot + ns > p.max_slot)) return;   // see below
    for (int s = 0; s < ns; ++s) {
      RaggedSeg g;
      g.req = (int32_t)r;
      g.tile = (int32_t)i;
      g.kt0 = (int32_t)((int64_t)nkt * s / ns);
      g.kt1 = (int32_t)((int64_t)nkt * (s + 1) / ns);
      g.slot = ns > 1 ? (int32_t)slot + s : -1;
      g.first = (int32_t)slot;
      g.parts = ns;
      g.pad = 0;
      p.segs[seg + s] = g;
    }
  };
  uint64_t base = 0;
  for (int64_t r0 = 0; r0 < p.rv.R; r0 += kPlanThreads) {
    const int64_t r = r0 + tid;
    const Request q = listed_request(p, r);
    const int64_t tiles = (q.q_len + p.pcta - 1) / p.pcta;
    uint64_t mine = 0;
    if (tiles <= 32)
      for (int64_t i = 0; i < tiles; ++i) mine += cuts(key_tiles(p, q, i));
    const unsigned bigs = __ballot_sync(0xffffffffu, tiles > 32);
    for (unsigned big = bigs; big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Request bq;
      bq.q0 = 0;
      bq.q_len = __shfl_sync(0xffffffffu, q.q_len, src);
      bq.seq = __shfl_sync(0xffffffffu, q.seq, src);
      const int64_t bt = __shfl_sync(0xffffffffu, tiles, src);
      uint64_t part = 0;
      for (int64_t i = lane; i < bt; i += 32) part += cuts(key_tiles(p, bq, i));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == src) mine = part;
    }
    uint64_t at = base + block_scan(mine, warp_tot, sum) - mine;
    base += sum;
    if (tiles <= 32)
      for (int64_t i = 0; i < tiles; ++i) {
        const int nkt = key_tiles(p, q, i);
        put(r, i, nkt, at);
        at += cuts(nkt);
      }
    for (unsigned big = bigs; big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Request bq;
      bq.q0 = 0;
      bq.q_len = __shfl_sync(0xffffffffu, q.q_len, src);
      bq.seq = __shfl_sync(0xffffffffu, q.seq, src);
      const int64_t bt = __shfl_sync(0xffffffffu, tiles, src);
      const int64_t br = __shfl_sync(0xffffffffu, r, src);
      uint64_t run = __shfl_sync(0xffffffffu, at, src);
      for (int64_t i0 = 0; i0 < bt; i0 += 32) {
        const int64_t i = i0 + lane;
        const int nkt = i < bt ? key_tiles(p, bq, i) : 0;
        const uint64_t own = i < bt ? cuts(nkt) : 0;
        uint64_t x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (i < bt) put(br, i, nkt, run + x - own);
        run += __shfl_sync(0xffffffffu, x, 31);
      }
    }
  }
  // the bounds hold for ascending offsets; a batch that breaks them is not run
  if (tid == 0) {
    const bool ok = (uint32_t)base <= (uint32_t)p.max_seg && (base >> 32) <= (uint64_t)p.max_slot;
    if (!ok) atomicOr(p.status, TQ_DEV_BAD_BATCH);
    *p.nseg = ok ? (int32_t)(uint32_t)base : 0;
  }
}

// Shape of one list's launch: head group, query positions and rows of a CTA,
// the bounds of the work list and its place in the workspace.
struct ListShape {
  bool used;
  int64_t q_lo, q_hi;
  int hc, pcta, rows, keys, G;
  int64_t wanted, max_seg, max_slot;
  size_t off_nseg, off_segs, off_arrived, off_ml, off_part;
};

struct AttendShape {
  bool tc;                                 // the wide list runs on tcgen05
  int64_t Hkv;
  ListShape few, wide;
  size_t bytes;
};

// Query rows of a request and KV head up to which the few-row kernel is taken.
constexpr int kFewRows = 64;

AttendShape attend_shape(const tq_geom* G, const tq_cache* c, const tq_attend_args* a) {
  AttendShape s = {};
  const int64_t R = a->batch.requests, N = a->q->shape[2], most = INT64_MAX;
  s.Hkv = c->streams / R;
  const int64_t g = a->q->shape[1] / s.Hkv;
  s.tc = prefill_tc_applies(G) && a->engine != 1;
  const bool can = attend_few_applies(G) && (a->engine == 0 || a->engine == 3);
  const int64_t few_q = a->engine == 3 ? most : tmax<int64_t>(kFewRows / g, 1);
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
    l.off_nseg = 68;
    finish(l);
  }
  s.bytes = off;
  return s;
}

}  // namespace

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
    p.segs = reinterpret_cast<RaggedSeg*>(base + l->off_segs);
    p.arrived = reinterpret_cast<int32_t*>(base + l->off_arrived);
    p.status = status;
    RaggedAttend& r = rg[lists++];
    r.rv = p.rv;
    r.plan.segs = p.segs;
    r.plan.nseg = p.nseg;
    r.plan.arrived = p.arrived;
    r.plan.ml = reinterpret_cast<float2*>(base + l->off_ml);
    r.plan.part = reinterpret_cast<float*>(base + l->off_part);
    r.plan.G = l->G;
    r.plan.rows = l->rows;
  }
  ragged_plan_kernel<<<lists, kPlanThreads, 0, st>>>(plan[0], plan[lists - 1]);
  if (check_launch("tq_attend_ragged/plan") != TQ_OK) return TQ_ERR_CUDA;
  if (s.few.used) {
    const int rc = launch_attend_few(G, t, c, a, rg[0], s.Hkv, s.few.hc, s.few.pcta, s.few.rows,
                                     s.few.max_seg * s.few.G, status, st);
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
