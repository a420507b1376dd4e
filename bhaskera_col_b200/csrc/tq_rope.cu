// tq_rope.cu — norm and rotation of query and key heads in one pass
// (tq_qk_rope): y = rotation(x / rms(x) * w) in fp32, rounded once.
#include "tq_internal.h"
#include "tq_ragged.cuh"

namespace tq {
namespace {

struct RopeSide {
  const void* x;
  void* y;
  int64_t xs[4], ys[4];
  int64_t H;
  int dtype;
  HeadXform f;
};

struct RopeParams {
  RopeSide side[2];             // q, k (H = 0: absent)
  int64_t B, T;
  int D;
  const void* pos; int pos64; int64_t ps[2];
  uint32_t* status;
};

constexpr int kRopeWarps = 8;

__device__ __forceinline__ int64_t load_pos(const void* pos, int pos64, int64_t i) {
  return pos64 ? __ldg(reinterpret_cast<const long long*>(pos) + i)
               : (int64_t)__ldg(reinterpret_cast<const int*>(pos) + i);
}

// Any type, stride, head size and rotary part: one warp per head vector, the
// vector staged in shared memory.
__global__ void __launch_bounds__(32 * kRopeWarps) rope_any_kernel(RopeParams p) {
  __shared__ float rows[kRopeWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* u = rows[warp];
  const int64_t Hs = p.side[0].H + p.side[1].H, total = p.B * p.T * Hs;
  for (int64_t i = blockIdx.x * (int64_t)kRopeWarps + warp; i < total;
       i += (int64_t)gridDim.x * kRopeWarps) {
    const int64_t tok = i / Hs, b = tok / p.T, t = tok % p.T;
    int64_t h = i % Hs;
    const int w = h >= p.side[0].H;
    if (w) h -= p.side[0].H;
    const RopeSide& s = p.side[w];
    const int64_t xb = b * s.xs[0] + h * s.xs[1] + t * s.xs[2];
    for (int c = lane; c < p.D; c += 32) u[c] = load_elem(s.x, s.dtype, xb + c * s.xs[3]);
    __syncwarp();
    int64_t row = 0;
    if (s.f.cos_sin)
      row = table_row(s.f, load_pos(p.pos, p.pos64, b * p.ps[0] + t * p.ps[1]), p.status);
    xform_row(u, p.D, s.f, row, lane);
    const int64_t yb = b * s.ys[0] + h * s.ys[1] + t * s.ys[2];
    for (int c = lane; c < p.D; c += 32) store_elem(s.y, s.dtype, yb + c * s.ys[3], u[c]);
    __syncwarp();
  }
}

}  // namespace

int launch_qk_rope(const tq_rope* rope, const tq_positions* pos, const tq_tensor4* const x[2],
                   const tq_tensor4* const y[2], const tq_head_norm* const norm[2],
                   uint32_t* status, cudaStream_t st) {
  RopeParams p;
  for (int w = 0; w < 2; ++w) {
    RopeSide& s = p.side[w];
    s.H = 0;
    if (!x[w]) continue;
    s.x = x[w]->data; s.y = y[w]->data; s.dtype = x[w]->dtype;
    for (int i = 0; i < 4; ++i) { s.xs[i] = x[w]->stride[i]; s.ys[i] = y[w]->stride[i]; }
    s.H = x[w]->shape[1];
    s.f = head_xform(rope, norm[w]);
    p.B = x[w]->shape[0];
    p.T = x[w]->shape[2];
    p.D = (int)x[w]->shape[3];
  }
  p.pos = pos ? pos->data : nullptr;
  p.pos64 = pos && pos->bits == 64;
  p.ps[0] = pos ? pos->stride[0] : 0;
  p.ps[1] = pos ? pos->stride[1] : 0;
  p.status = status;
  const int64_t total = p.B * p.T * (p.side[0].H + p.side[1].H);
  if (total == 0) return TQ_OK;
  const int64_t blocks = (total + kRopeWarps - 1) / kRopeWarps;
  rope_any_kernel<<<(unsigned)tmin<int64_t>(blocks, 16 * device_sm_count()), 32 * kRopeWarps, 0,
                    st>>>(p);
  return check_launch("tq_qk_rope");
}

}  // namespace tq
