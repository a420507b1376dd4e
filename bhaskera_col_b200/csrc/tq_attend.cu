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
#include "tq_internal.h"
#include "tq_ragged.cuh"

namespace tq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kWaves = 3;                  // segments wanted per SM
constexpr int kMinKeys = 512;              // shortest segment worth a CTA's set-up

struct PlanParams {
  RaggedView rv;
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
__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(PlanParams p) {
  __shared__ uint64_t warp_tot[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < p.max_slot * p.G; i += kPlanThreads) p.arrived[i] = 0;
  // f(request, tile, lane's turn) for every tile of this thread's request
  uint64_t total = 0, sum = 0;
  for (int64_t r0 = 0; r0 < p.rv.R; r0 += kPlanThreads) {
    const int64_t r = r0 + tid;
    Request q = {};
    if (r < p.rv.R) q = request_at(p.rv, r);
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
    Request q = {};
    if (r < p.rv.R) q = request_at(p.rv, r);
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

// Shape of the launch: head group, query positions and rows of a CTA, and the
// bounds of the work list; the workspace follows from it.
struct AttendShape {
  int engine, hc, pcta, rows, keys, G;
  int64_t Hkv, wanted;
  int64_t max_seg, max_slot;
  size_t off_segs, off_arrived, off_ml, off_part, bytes;
};

AttendShape attend_shape(const tq_geom* G, const tq_cache* c, const tq_attend_args* a) {
  AttendShape s = {};
  const int64_t R = a->batch.requests, N = a->q->shape[2];
  s.Hkv = c->streams / R;
  const int64_t g = a->q->shape[1] / s.Hkv;
  s.engine = 1;
  s.hc = g % 8 == 0 ? 8 : g % 4 == 0 ? 4 : g % 2 == 0 ? 2 : 1;
  s.rows = 128;
  s.keys = 64;
  s.pcta = s.rows / s.hc;
  s.G = (int)(s.Hkv * (g / s.hc));
  s.wanted = (int64_t)kWaves * device_sm_count();
  // tiles: one per started block of positions; L cuts off at most wanted / G
  // segments beyond them, and a cut tile has at most twice its extra ones
  const int64_t extra = s.wanted / s.G + 1;
  s.max_seg = N / s.pcta + R + extra;
  s.max_slot = 2 * extra;
  size_t off = 256;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) & ~(size_t)255;
    return at;
  };
  s.off_segs = take(s.max_seg * sizeof(RaggedSeg));
  s.off_arrived = take(s.max_slot * s.G * 4);
  s.off_ml = take((size_t)s.max_slot * s.G * s.rows * 8);
  s.off_part = take((size_t)s.max_slot * s.G * s.rows * G->head_dim * 4);
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
  PlanParams p;
  p.rv = ragged_view(&a->batch, a->q->shape[2], c);
  p.pcta = s.pcta;
  p.keys = s.keys;
  p.causal = a->causal;
  p.G = s.G;
  p.wanted = s.wanted;
  p.min_tiles = kMinKeys / s.keys;
  p.max_seg = (int)s.max_seg;
  p.max_slot = (int)s.max_slot;
  p.nseg = reinterpret_cast<int32_t*>(base + 64);   // below: the decode's status word
  p.segs = reinterpret_cast<RaggedSeg*>(base + s.off_segs);
  p.arrived = reinterpret_cast<int32_t*>(base + s.off_arrived);
  p.status = status;
  ragged_plan_kernel<<<1, kPlanThreads, 0, st>>>(p);
  if (check_launch("tq_attend_ragged/plan") != TQ_OK) return TQ_ERR_CUDA;
  RaggedAttend rg;
  rg.rv = p.rv;
  rg.plan.segs = p.segs;
  rg.plan.nseg = p.nseg;
  rg.plan.arrived = p.arrived;
  rg.plan.ml = reinterpret_cast<float2*>(base + s.off_ml);
  rg.plan.part = reinterpret_cast<float*>(base + s.off_part);
  rg.plan.G = s.G;
  rg.plan.rows = s.rows;
  return launch_attend_mma(G, t, c, a, rg, s.Hkv, s.hc, s.max_seg * s.G, status, st);
}

}  // namespace tq
