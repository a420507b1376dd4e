// tq_ragged.cuh — ragged batches: requests of different lengths flattened into
// one run of tokens (token i of request r is row q_start[r] + i and sits at
// position seq_lens[r] - q_len + i of its request), and the norm + rotation
// of a head vector that the serving operators apply on the way.
#pragma once

#include "tq_common.cuh"

namespace tq {

// ---------------------------------------------------------------------------
// Requests
// ---------------------------------------------------------------------------
struct RaggedView {
  const int32_t* q_start;     // [R + 1]
  const int32_t* seq_lens;    // [R]
  int64_t R, N, cap;          // requests, rows of the flattened tensors, tokens a request can hold
};

struct Request {
  int64_t q0, q_len, seq;     // first row, rows, tokens in the cache (new ones included)
  int64_t base;               // position of the first row
};

// Do the offsets ascend within [0, N]?  Thread tid of n looks at every n-th request;
// whoever sees one that does not sets TQ_DEV_BAD_BATCH, and the block agrees not to
// run.  The first request's offsets are loaded when the check is made, so that other
// loads hide their way (0.5 us of a launch of few tokens).
struct OffsetCheck {
  int a, b;
  __device__ __forceinline__ OffsetCheck(const RaggedView& v, int tid) : a(0), b(0) {
    if (tid < v.R) {
      a = __ldg(v.q_start + tid);
      b = __ldg(v.q_start + tid + 1);
    }
  }
  __device__ __forceinline__ bool fails(const RaggedView& v, int tid, int n, uint32_t* status) const {
    bool bad = a < 0 || a > b || b > v.N;
    for (int64_t r = (int64_t)tid + n; r < v.R; r += n) {
      const int c = __ldg(v.q_start + r), d = __ldg(v.q_start + r + 1);
      bad = bad || c < 0 || c > d || d > v.N;
    }
    if (bad) atomicOr(status, TQ_DEV_BAD_BATCH);
    return bad;
  }
};

// Request r, with offsets outside the tensors cut to them: a wrong offset
// never leads outside memory.
__device__ __forceinline__ Request request_at(const RaggedView& v, int64_t r) {
  Request q;
  const int64_t a = __ldg(v.q_start + r), b = __ldg(v.q_start + r + 1), s = __ldg(v.seq_lens + r);
  q.q0 = tmin(tmax<int64_t>(a, 0), v.N);
  q.q_len = tmax<int64_t>(tmin(b, v.N) - q.q0, 0);
  q.seq = tmin(tmax<int64_t>(s, 0), v.cap);
  // of the length as it is, so that rows keep their places (from 2^30 - 64 on, where no
  // pages reach, all places are one: sums with rows stay within 32 bits)
  q.base = tmin<int64_t>(tmax<int64_t>(s, 0) - q.q_len, (1 << 30) - 64);
  return q;
}

// The request that holds row n: the last r with q_start[r] <= n, or -1 for a
// row outside every request.
__device__ __forceinline__ int64_t request_of(const RaggedView& v, int64_t n) {
  int64_t lo = 0, hi = v.R;                 // q_start[lo] <= n < q_start[hi] at the end
  if (n < __ldg(v.q_start) || n >= __ldg(v.q_start + v.R)) return -1;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(v.q_start + mid) <= n) lo = mid; else hi = mid;
  }
  return lo;
}

// Where row n lives: its request and its position there; false for a row
// outside every request or a position outside [0, cap).
__device__ __forceinline__ bool locate_row(const RaggedView& v, int64_t n, int64_t& r,
                                           int64_t& pos) {
  r = request_of(v, n);
  if (r < 0) return false;
  pos = (int64_t)__ldg(v.seq_lens + r) - __ldg(v.q_start + r + 1) + n;
  return pos >= 0 && pos < v.cap;
}

// ---------------------------------------------------------------------------
// x -> rotation(rms_norm(x)) of one head vector
// ---------------------------------------------------------------------------
// Position axes: pair i turns by the token's position on axis `of`[i], 2 bits a pair;
// n = 0: one axis.
struct AxisMap {
  int n;
  int64_t stride;             // of positions, from axis to axis
  uint32_t of[8];
  __device__ __forceinline__ int axis(int pair) const { return (of[pair >> 4] >> (2 * (pair & 15))) & 3; }
};

struct HeadXform {
  const float* cos_sin;       // [positions][rot]: cosines, then sines; NULL: no rotation
  int64_t positions;
  int rot, interleaved;
  const void* weight;         // [D] or NULL: no norm
  int w_dtype;
  float eps, w_offset;
  AxisMap axes;
};

__device__ __forceinline__ int64_t load_pos(const void* pos, int pos64, int64_t i) {
  return pos64 ? __ldg(reinterpret_cast<const long long*>(pos) + i)
               : (int64_t)__ldg(reinterpret_cast<const int*>(pos) + i);
}

// Row index of a position in the rotation table; positions outside it take
// row 0 and set TQ_DEV_BAD_POSITION.
__device__ __forceinline__ int64_t table_row(const HeadXform& f, int64_t pos, uint32_t* status) {
  if (pos >= 0 && pos < f.positions) return pos;
  atomicOr(status, TQ_DEV_BAD_POSITION);
  return 0;
}

// One warp, the vector in shared memory (u[0..D), already visible to the
// warp): norm and rotation in fp32, in place; visible to the warp on return.
// row_of(i) is the table's row for pair i.
template <class RowOf>
__device__ __forceinline__ void xform_row(float* u, int D, const HeadXform& f, int lane,
                                          RowOf row_of) {
  if (f.weight) {
    float ss = 0.f;
    for (int c = lane; c < D; c += 32) ss = fmaf(u[c], u[c], ss);
    const float inv = 1.f / sqrtf(warp_sum(ss) / (float)D + f.eps);
    for (int c = lane; c < D; c += 32)
      u[c] = u[c] * inv * (load_elem(f.weight, f.w_dtype, c) + f.w_offset);
    __syncwarp();
  }
  if (f.cos_sin) {
    const int half = f.rot / 2;
    for (int i = lane; i < half; i += 32) {
      const float* cs = f.cos_sin + row_of(i) * f.rot;
      const int ia = f.interleaved ? 2 * i : i, ib = f.interleaved ? 2 * i + 1 : half + i;
      const float a = u[ia], b = u[ib], c = __ldg(cs + i), s = __ldg(cs + half + i);
      u[ia] = a * c - b * s;
      u[ib] = b * c + a * s;
    }
    __syncwarp();
  }
}

// The same at one row for all pairs, or at the token's positions pos[at], a row an axis.
__device__ __forceinline__ void xform_row(float* u, int D, const HeadXform& f, int64_t row,
                                          int lane) {
  xform_row(u, D, f, lane, [&](int) { return row; });
}
__device__ __forceinline__ void xform_axes(float* u, int D, const HeadXform& f, const void* pos,
                                           int pos64, int64_t at, uint32_t* status, int lane) {
  xform_row(u, D, f, lane, [&](int i) {
    return table_row(f, load_pos(pos, pos64, at + f.axes.axis(i) * f.axes.stride), status);
  });
}

// cos and sin of N neighbouring pairs from pair i0 on (a multiple of N), each from its
// own axis' row of the table; row_of(a) is axis a's.  An axis that none of the pairs
// follows is not read.  The table's row and its halves are N-aligned.
template <int N, class RowOf>
__device__ __forceinline__ void load_axes(float (&cs)[N], float (&sn)[N], const HeadXform& f, int i0,
                                          RowOf row_of) {
  const int half = f.rot / 2;
  const uint32_t of = f.axes.of[i0 >> 4] >> (2 * (i0 & 15));
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < N; ++e) any = any || ((of >> (2 * e)) & 3u) == (uint32_t)a;
    if (a >= f.axes.n || !any) continue;
    const float* tab = f.cos_sin + row_of(a) * f.rot + i0;
    float c[N], s[N];
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(tab + e));
        const float4 y = __ldg(reinterpret_cast<const float4*>(tab + half + e));
        c[e] = x.x; c[e + 1] = x.y; c[e + 2] = x.z; c[e + 3] = x.w;
        s[e] = y.x; s[e + 1] = y.y; s[e + 2] = y.z; s[e + 3] = y.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        c[e] = __ldg(tab + e);
        s[e] = __ldg(tab + half + e);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool mine = ((of >> (2 * e)) & 3u) == (uint32_t)a;
      cs[e] = mine ? c[e] : cs[e];
      sn[e] = mine ? s[e] : sn[e];
    }
  }
}

// ---------------------------------------------------------------------------
// Work list of the ragged attention: every (request, block of query
// positions) is one tile; its key tiles are cut into segments, one CTA each
// (times the head groups).  Built on the device by ragged_plan_kernel.
// ---------------------------------------------------------------------------
struct RaggedSeg {
  int32_t req, tile;          // request, block of query positions
  int32_t kt0, kt1;           // key tiles
  int32_t slot;               // partial slot of this segment, -1: it is the tile's only one
  int32_t first, parts;       // the tile's first slot and its segments
  int32_t pad;
};

struct RaggedPlan {
  const RaggedSeg* segs;
  const int32_t* nseg;
  int32_t* next;              // next (segment, head group) to be taken
  int32_t* arrived;           // [slots][G] finished segments of the tile, at its first slot
  float* part;                // [slots][G][rows][D] partial outputs
  float2* ml;                 // [slots][G][rows] running max (log2) and sum
  int G;                      // head groups: KV heads x chunks of their query heads
  int rows;                   // query rows of a CTA
};

// Which query heads, streams and columns a head group stands for.  Plain attention: KV
// head kvh, its g query heads, columns of the head.  Differential attention works on
// 2 H heads in pairs, head v = 2 h + m (map m of pair h), which lie in q as they are or
// (halves) the first maps before the second ones.  own: maps with keys of their own,
// kvh = (p, m, j): the heads of map m of KV pair p over the keys of its head m and the
// values of its head j, columns D j of the result.
struct HeadView {
  int own, halves;
  int H, P;                   // pairs of query heads; pairs of KV heads (own)
  int g;                      // heads of a group's KV head, all chunks
  int streams;                // KV heads of a request in the cache
  __device__ __forceinline__ int kv_pair(int p, int m) const { return halves ? m * P + p : 2 * p + m; }
  __device__ __forceinline__ int key_head(int kvh) const { return own ? kv_pair(kvh >> 2, (kvh >> 1) & 1) : kvh; }
  __device__ __forceinline__ int value_head(int kvh) const { return own ? kv_pair(kvh >> 2, kvh & 1) : kvh; }
  // head i of the group, and its place in q
  __device__ __forceinline__ int head(int kvh, int i) const {
    return own ? 2 * ((kvh >> 2) * g + i) + ((kvh >> 1) & 1) : kvh * g + i;
  }
  __device__ __forceinline__ int in_q(int v) const { return halves ? (v >> 1) + (v & 1) * H : v; }
  // first column of the head's result
  __device__ __forceinline__ int column(int kvh, int D) const { return own ? (kvh & 1) * D : 0; }
};

struct RaggedAttend {
  RaggedView rv;
  RaggedPlan plan;
  HeadView hv;
};

// One CTA's share of the work list.
struct SegWork {
  Request rq;
  RaggedSeg seg;
  int group;
};

// Item `i` of the list (segment x head group); false past its end.
__device__ __forceinline__ bool take_segment(const RaggedAttend& a, unsigned i, SegWork& w) {
  const int si = (int)(i / (unsigned)a.plan.G);
  w.group = (int)(i % (unsigned)a.plan.G);
  if (si >= *a.plan.nseg) return false;
  w.seg = a.plan.segs[si];
  w.rq = request_at(a.rv, w.seg.req);
  return true;
}

// Partial results of one query row of a split tile.
__device__ __forceinline__ int64_t part_row(const RaggedPlan& pl, int slot, int group, int row) {
  return ((int64_t)slot * pl.G + group) * pl.rows + row;
}

// Called by every thread of a CTA that has stored its part of a split tile:
// true for the tile's last CTA, which then sees the parts of all others.
__device__ __forceinline__ bool last_of_tile(const RaggedPlan& pl, const SegWork& w, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const int done = atomicAdd(pl.arrived + (int64_t)w.seg.first * pl.G + w.group, 1);
    *flag = done == w.seg.parts - 1;
    __threadfence();
  }
  __syncthreads();
  return *flag != 0;
}

// The last CTA of a split tile joins its partials (out / l and {m, l}),
//   M = max_s m_s, w_s = l_s 2^(m_s - M), out = sum_s w_s out_s / sum_s w_s,
// in slot order whatever the order of arrival, one warp per row.  `row_out(row)`
// gives the element offset of a row's output, or -1 for a row without a query.
// A NaN sum (see tq_attend_ragged) makes the row NaN.
template <int D, class RowOut>
__device__ __forceinline__ void join_partials(const RaggedPlan& pl, const SegWork& w, int nwarps,
                                              void* out, int o_dtype, int64_t o_stride,
                                              int* last_flag, RowOut row_out) {
  if (!last_of_tile(pl, w, last_flag)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int row = warp; row < pl.rows; row += nwarps) {
    const int64_t at = row_out(row);
    if (at < 0) continue;
    float M = -INFINITY;
    for (int s = lane; s < w.seg.parts; s += 32) {
      const float2 ml = __ldcg(pl.ml + part_row(pl, w.seg.first + s, w.group, row));
      if (ml.y > 0.f) M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float sum = 0.f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
    for (int s = 0; s < w.seg.parts; ++s) {
      const int64_t pr = part_row(pl, w.seg.first + s, w.group, row);
      const float2 ml = __ldcg(pl.ml + pr);
      if (ml.y == 0.f) continue;                    // no key seen in this segment
      const float ws = ml.y * fast_exp2(ml.x - M);
      sum += ws;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        acc[i] = fmaf(ws, __ldcg(pl.part + pr * D + 32 * i + lane), acc[i]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      store_elem(out, o_dtype, at + (int64_t)(32 * i + lane) * o_stride, acc[i] * inv);
  }
}

}  // namespace tq
