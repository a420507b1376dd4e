// tq_ragged.cu — ragged append (norm -> rotate position -> quantise -> pack)
// and ragged read-back on CUDA cores, for every supported geometry.
//
// The math per vector is tq_append's (tq_vec.cuh: fp32 norm n, u = x /
// max(n, 1e-8), y = u R^T summed in ascending order, code = #{boundaries < y})
// and tq_dequantize's (x = (c[code] R) n).  Bound by the rotation's fp32 products
// (D^2 a vector): the shapes of the tensor-core kernels took 3 to 16 times as long
// here (single tokens 43 us against 27, 17,971 tokens read back 877 against 51).
#include "tq_internal.h"
#include "tq_ragged.cuh"
#include "tq_vec.cuh"

namespace tq {

HeadXform head_xform(const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm) {
  HeadXform f = {};
  if (rope && axes) {
    f.axes.n = axes->axes;
    f.axes.stride = axes->stride;
    for (int i = 0; i < rope->rot_dim / 2; ++i)
      f.axes.of[i >> 4] |= (uint32_t)axes->axis[i] << (2 * (i & 15));
  }
  if (rope) {
    f.cos_sin = rope->cos_sin;
    f.positions = rope->positions;
    f.rot = rope->rot_dim;
    f.interleaved = rope->interleaved;
  }
  if (norm) {
    f.weight = norm->weight;
    f.w_dtype = norm->dtype;
    f.eps = norm->eps;
    f.w_offset = norm->offset;
  }
  return f;
}

RaggedView ragged_view(const tq_ragged* b, int64_t N, const tq_cache* c) {
  RaggedView v;
  v.q_start = b->q_start;
  v.seq_lens = b->seq_lens;
  v.R = b->requests;
  v.N = N;
  v.cap = c->pages_per_stream * kPageTokens;
  return v;
}

namespace {

constexpr int kVecs = 16;                // vectors per tile
constexpr int kThreadsR = 256;

struct RaggedKV {
  PageGeom g;
  const float* cent[2];
  const float* bnd[2];
  const float* R;                        // append: R^T, read-back: R (row-major)
  uint8_t* pages;
  PageMap pm;
  uint32_t* status;
  RaggedView rv;
  int64_t H;
  const void* x[2];                      // append: inputs; read-back: outputs (NULL: absent)
  int dtype[2];
  int64_t stride[2][3];                  // head, row, dim
  HeadXform f;                           // of K (append)
  const void* pos; int pos64; int64_t pos_stride;
};

// Row and head of vector i (token-major), its page row: false when it has none.
__device__ __forceinline__ bool vec_slot(const RaggedKV& p, int64_t i, int64_t& n, int64_t& h,
                                         int64_t& pos, uint8_t*& page, bool& inside) {
  n = i / p.H;
  h = i % p.H;
  int64_t r;
  inside = request_of(p.rv, n) >= 0;
  if (!locate_row(p.rv, n, r, pos)) {
    if (inside) atomicOr(p.status, TQ_DEV_BAD_POSITION);
    return false;
  }
  bool ok;
  const int64_t ps = page_slot(p.pm, r * p.H + h, pos / kPageTokens, ok);
  if (!ok) atomicOr(p.status, TQ_DEV_BAD_BLOCK);
  page = p.pages + ps * (int64_t)p.g.page_bytes;
  return ok;
}

template <int D>
__global__ void __launch_bounds__(kThreadsR) append_ragged_kernel(RaggedKV p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int which = blockIdx.y;           // 0: K, 1: V
  const PageGeom& g = p.g;
  const int bits = which == 0 ? g.kb : g.vb, nb = (1 << bits) - 1;
  float* RT = reinterpret_cast<float*>(smem);                  // [D][D]
  float* u = RT + D * D;                                       // [kVecs][D]
  float* bb = u + kVecs * D;                                   // [256]
  float* nrm = bb + 256;                                       // [kVecs]
  uint8_t** page = reinterpret_cast<uint8_t**>(nrm + kVecs);   // [kVecs] page or NULL
  int* slot = reinterpret_cast<int*>(page + kVecs);            // [kVecs] token in the page
  uint8_t* code = reinterpret_cast<uint8_t*>(slot + kVecs);    // [kVecs][D]
  int16_t* ord = reinterpret_cast<int16_t*>(code + kVecs * D); // [D]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  stage_async(RT, p.R, D * D * 4, tid, kThreadsR);
  cp_async_wait_all();
  for (int i = tid; i < nb; i += kThreadsR) bb[i] = p.bnd[which][i];
  if (which == 0) build_orders(ord, nullptr, nullptr, D, tid, kThreadsR);
  else build_orders(nullptr, ord, nullptr, D, tid, kThreadsR);
  if (__syncthreads_or(OffsetCheck(p.rv, tid).fails(p.rv, tid, kThreadsR, p.status))) return;
  const int rowbytes = which == 0 ? g.krow : g.vrow;
  const int sec = which == 0 ? g.off_k : g.off_v, nsec = which == 0 ? g.off_kn : g.off_vn;
  const int64_t nvec = p.rv.N * p.H;
  for (int64_t v0 = (int64_t)blockIdx.x * kVecs; v0 < nvec; v0 += (int64_t)gridDim.x * kVecs) {
    const int nv = (int)tmin<int64_t>(kVecs, nvec - v0);
    for (int v = warp; v < nv; v += kThreadsR / 32) {
      int64_t n = 0, h = 0, pos = 0;
      uint8_t* pg = nullptr;
      bool inside;
      const bool ok = vec_slot(p, v0 + v, n, h, pos, pg, inside);
      if (lane == 0) {
        page[v] = ok ? pg : nullptr;
        slot[v] = (int)(pos % kPageTokens);
      }
      if (!ok) continue;
      float* uv = u + v * D;
      const int64_t base = h * p.stride[which][0] + n * p.stride[which][1];
      for (int c = lane; c < D; c += 32)
        uv[c] = load_elem(p.x[which], p.dtype[which], base + c * p.stride[which][2]);
      __syncwarp();
      if (which == 0 && (p.f.weight || p.f.cos_sin)) {
        if (p.f.axes.n) {
          xform_axes(uv, D, p.f, p.pos, p.pos64, n * p.pos_stride, p.status, lane);
        } else {
          int64_t row = 0;
          if (p.f.cos_sin)
            row = table_row(p.f, p.pos ? load_pos(p.pos, p.pos64, n * p.pos_stride) : pos, p.status);
          xform_row(uv, D, p.f, row, lane);
        }
      }
      float ss = 0.f;
      for (int c = lane; c < D; c += 32) ss = fmaf(uv[c], uv[c], ss);
      const float nr = sqrtf(warp_sum(ss)), den = fmaxf(nr, 1e-8f);
      for (int c = lane; c < D; c += 32) uv[c] = uv[c] / den;
      if (lane == 0) nrm[v] = nr;
    }
    __syncthreads();
    for (int i = tid; i < nv * D; i += kThreadsR) {
      const int v = i / D, j = i % D;
      code[i] = page[v] ? (uint8_t)bucketize_lt(bb, nb, rot_coord(u + v * D, RT, j, D)) : 0;
    }
    __syncthreads();
    const int words = rowbytes / 4;
    for (int i = tid; i < nv * words; i += kThreadsR) {
      const int v = i / words, w = i % words;
      if (page[v])
        reinterpret_cast<uint32_t*>(page[v] + sec + slot[v] * rowbytes)[w] =
            pack_word(code + v * D, ord, bits, w, D);
    }
    for (int v = tid; v < nv; v += kThreadsR)
      if (page[v]) reinterpret_cast<__half*>(page[v] + nsec)[slot[v]] = __float2half_rn(nrm[v]);
    __syncthreads();
  }
}

template <int D>
size_t append_ragged_smem() {
  return (size_t)(D * D + kVecs * D + 256 + kVecs) * 4 + kVecs * (8 + 4 + D) + 2 * D;
}

template <int D>
__global__ void __launch_bounds__(kThreadsR) read_ragged_kernel(RaggedKV p) {
  __shared__ float cv[kVecs][D];
  __shared__ float nr[kVecs];
  __shared__ int state[kVecs];            // 0: leave the row, 1: zero it, 2: write it
  const int which = blockIdx.y;
  if (!p.x[which]) return;
  const PageGeom& g = p.g;
  const int bits = which == 0 ? g.kb : g.vb;
  const int rowbytes = which == 0 ? g.krow : g.vrow;
  const int sec = which == 0 ? g.off_k : g.off_v, nsec = which == 0 ? g.off_kn : g.off_vn;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t nvec = p.rv.N * p.H;
  if (__syncthreads_or(OffsetCheck(p.rv, tid).fails(p.rv, tid, kThreadsR, p.status))) return;
  for (int64_t v0 = (int64_t)blockIdx.x * kVecs; v0 < nvec; v0 += (int64_t)gridDim.x * kVecs) {
    const int nv = (int)tmin<int64_t>(kVecs, nvec - v0);
    for (int v = warp; v < nv; v += kThreadsR / 32) {
      int64_t n = 0, h = 0, pos = 0;
      uint8_t* pg = nullptr;
      bool inside;
      const bool ok = vec_slot(p, v0 + v, n, h, pos, pg, inside);
      if (lane == 0) state[v] = ok ? 2 : inside ? 1 : 0;
      if (!ok) continue;
      const int sl = (int)(pos % kPageTokens);
      const uint32_t* row = reinterpret_cast<const uint32_t*>(pg + sec + sl * rowbytes);
      for (int c = lane; c < D; c += 32) {
        const int bo = (which == 0 ? k_pos_of(c, D) : v_pos_of(c, D)) * bits, sh = bo & 31;
        uint32_t w = __ldg(row + (bo >> 5)) >> sh;
        if (sh + bits > 32) w |= __ldg(row + (bo >> 5) + 1) << (32 - sh);
        cv[v][c] = __ldg(p.cent[which] + (w & ((1u << bits) - 1u)));
      }
      if (lane == 0) nr[v] = __half2float(reinterpret_cast<const __half*>(pg + nsec)[sl]);
    }
    __syncthreads();
    for (int i = tid; i < nv * D; i += kThreadsR) {
      const int v = i / D, j = i % D;
      if (state[v] == 0) continue;
      float acc = 0.f;
      if (state[v] == 2) {
        for (int k = 0; k < D; ++k) acc = fmaf(cv[v][k], __ldg(p.R + k * D + j), acc);
        acc *= nr[v];
      }
      const int64_t n = (v0 + v) / p.H, h = (v0 + v) % p.H;
      store_elem(const_cast<void*>(p.x[which]), p.dtype[which],
                 h * p.stride[which][0] + n * p.stride[which][1] + j * p.stride[which][2], acc);
    }
    __syncthreads();
  }
}

RaggedKV ragged_kv(const tq_geom* G, const tq_tables* t, const tq_cache* c, const tq_tensor4* k,
                   const tq_tensor4* v, const tq_ragged* batch) {
  RaggedKV p = {};
  p.g = make_geom(G->head_dim, G->key_bits, G->value_bits, G->qjl);
  p.cent[0] = t->k_centroids; p.cent[1] = t->v_centroids;
  p.bnd[0] = t->k_boundaries; p.bnd[1] = t->v_boundaries;
  p.pages = c->pages;
  p.pm = page_map(c);
  const tq_tensor4* x[2] = {k, v};
  for (int w = 0; w < 2; ++w) {
    if (!x[w]) continue;
    p.x[w] = x[w]->data;
    p.dtype[w] = x[w]->dtype;
    for (int i = 0; i < 3; ++i) p.stride[w][i] = x[w]->stride[i + 1];
    p.H = x[w]->shape[1];
    p.rv = ragged_view(batch, x[w]->shape[2], c);
  }
  return p;
}

}  // namespace

int launch_append_ragged(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                         const tq_tensor4* k, const tq_tensor4* v, const tq_ragged* batch,
                         const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm,
                         const tq_positions* pos, uint32_t* status, cudaStream_t st) {
  if (!pos) axes = nullptr;                                // every axis at the token's position
  RaggedKV p = ragged_kv(G, t, c, k, v, batch);
  p.R = t->rot_t;
  p.status = status;
  p.f = head_xform(rope, axes, norm);
  p.pos = pos ? pos->data : nullptr;
  p.pos64 = pos && pos->bits == 64;
  p.pos_stride = pos ? pos->stride[1] : 0;
  const int64_t nvec = p.rv.N * p.H;
  if (nvec == 0) return TQ_OK;
  if (const int rc = launch_append_ragged_tc(G, t, c, k, v, batch, rope, axes, norm, pos, status, st); rc != 1)
    return rc;
  const int D = G->head_dim;
  const size_t smem = D == 32 ? append_ragged_smem<32>() : D == 64 ? append_ragged_smem<64>()
                    : D == 96 ? append_ragged_smem<96>() : append_ragged_smem<128>();
  void (*fn)(RaggedKV) = D == 32 ? append_ragged_kernel<32> : D == 64 ? append_ragged_kernel<64>
                       : D == 96 ? append_ragged_kernel<96> : append_ragged_kernel<128>;
  if (set_smem_attr((const void*)fn, smem) != TQ_OK) return TQ_ERR_CUDA;
  const int64_t tiles = (nvec + kVecs - 1) / kVecs;
  const int64_t fit = (int64_t)device_sm_count() * occupancy((const void*)fn, kThreadsR, smem);
  fn<<<dim3((unsigned)tmin(tiles, fit), 2), kThreadsR, smem, st>>>(p);
  return check_launch("tq_append_ragged");
}

int launch_dequant_ragged(const tq_geom* G, const tq_tables* t, const tq_cache* c,
                          const tq_ragged* batch, const tq_tensor4* ko, const tq_tensor4* vo,
                          uint32_t* status, cudaStream_t st) {
  RaggedKV p = ragged_kv(G, t, c, ko, vo, batch);
  p.R = t->rot;
  p.status = status;
  const int64_t nvec = p.rv.N * p.H;
  if (nvec == 0) return TQ_OK;
  if (const int rc = launch_dequant_ragged_tc(G, t, c, batch, ko, vo, status, st); rc != 1) return rc;
  const int D = G->head_dim;
  void (*fn)(RaggedKV) = D == 32 ? read_ragged_kernel<32> : D == 64 ? read_ragged_kernel<64>
                       : D == 96 ? read_ragged_kernel<96> : read_ragged_kernel<128>;
  const int64_t tiles = (nvec + kVecs - 1) / kVecs;
  fn<<<dim3((unsigned)tmin<int64_t>(tiles, 16 * device_sm_count()), 2), kThreadsR, 0, st>>>(p);
  return check_launch("tq_dequantize_ragged");
}

}  // namespace tq
