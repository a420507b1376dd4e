// tq_internal.h — host-side glue shared by the .cu translation units.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tq_b200.h"

namespace tq {

// Thread-local error message (tq_last_error).
void set_error(const char* fmt, ...);
// Returns TQ_OK, or TQ_ERR_CUDA with the launch error recorded.
int check_launch(const char* what);
// Same for the return code of an explicit launch (cudaLaunchKernelEx).
int launch_result(cudaError_t e, const char* what);
int set_smem_attr(const void* kernel, size_t bytes);
int device_sm_count();
// Resident CTAs per SM for a kernel (cached per device).
int occupancy(const void* kernel, int threads, size_t smem);

int launch_quantize_rotated(const float* y, int64_t n, const float* b, int nb,
                            int16_t* codes, cudaStream_t st);
int launch_append(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                  const tq_tensor4* k, const tq_tensor4* v, int64_t pos,
                  cudaStream_t st);
// Tensor-core append (head_dim 128, bf16 inputs, no QJL): TQ_OK when it ran,
// 1 when it does not apply (the caller uses the CUDA-core kernel), or an error.
int launch_append_tc(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                     const tq_tensor4* k, const tq_tensor4* v, int64_t pos, cudaStream_t st);
bool append_tc_applies(const tq_geom* g, const tq_tables* t, const tq_tensor4* k,
                       const tq_tensor4* v);
int read_tc_status(uint32_t* out, cudaStream_t st);
// Device address of the library status word read by tq_device_status.
uint32_t* device_status_word();
bool prefill_supported(int D, int kb, int vb);
// tcgen05 prefill attention (tq_prefill_tc.cu): TQ_OK when it ran, 1 when it
// does not apply (the caller uses the mma.sync kernel), or an error.
int launch_prefill_tc(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                      const tq_prefill_args* a, uint32_t* status, cudaStream_t st);
bool prefill_tc_applies(const tq_geom* g);
int launch_prefill(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                   const tq_prefill_args* a, uint32_t* status, cudaStream_t st);
int launch_dequant(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                   int64_t t0, int64_t t1, const tq_tensor4* ko, const tq_tensor4* vo,
                   cudaStream_t st);
size_t decode_workspace_bytes(const tq_geom* g, const tq_cache* c,
                              const tq_decode_args* a);
// The new token of a decode step (tq_decode_step): stored at `pos` by the
// query-preparation kernel before attention.
struct StepInput {
  const tq_tensor4* k;
  const tq_tensor4* v;
  int64_t pos;
};
int launch_decode(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                  const tq_decode_args* a, void* ws, size_t ws_bytes, cudaStream_t st,
                  const StepInput* step = nullptr);

// Serving operators on ragged batches (tq_rope.cu, tq_ragged.cu, tq_attend.cu).
struct HeadXform;
struct RaggedView;
struct RaggedAttend;
HeadXform head_xform(const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm);
RaggedView ragged_view(const tq_ragged* b, int64_t N, const tq_cache* c);
int launch_qk_rope(const tq_rope* rope, const tq_rope_axes* axes, const tq_positions* pos, const tq_tensor4* const x[2],
                   const tq_tensor4* const y[2], const tq_head_norm* const norm[2],
                   uint32_t* status, cudaStream_t st);
int launch_residual_norm(const tq_residual_norm_args* a, cudaStream_t st);
int launch_append_ragged(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                         const tq_tensor4* k, const tq_tensor4* v, const tq_ragged* batch,
                         const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm,
                         const tq_positions* pos, uint32_t* status, cudaStream_t st);
int launch_dequant_ragged(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                          const tq_ragged* batch, const tq_tensor4* ko, const tq_tensor4* vo,
                          uint32_t* status, cudaStream_t st);
// The tensor-core forms (tq_ragged_tc.cu): TQ_OK when they ran, 1 when they do
// not apply (the caller runs the CUDA-core kernels), or an error.
int launch_append_ragged_tc(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                            const tq_tensor4* k, const tq_tensor4* v, const tq_ragged* batch,
                            const tq_rope* rope, const tq_rope_axes* axes, const tq_head_norm* norm,
                            const tq_positions* pos, uint32_t* status, cudaStream_t st);
int launch_dequant_ragged_tc(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                             const tq_ragged* batch, const tq_tensor4* ko, const tq_tensor4* vo,
                             uint32_t* status, cudaStream_t st);
size_t attend_ragged_workspace(const tq_geom* g, const tq_cache* c, const tq_attend_args* a);
int launch_attend_ragged(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                         const tq_attend_args* a, void* ws, uint32_t* status, cudaStream_t st);
// Differential attention: a workspace of 0 bytes where no kernel applies.
bool attend_pair_applies(const tq_geom* g);
int launch_attend_pair(const tq_geom* g, const tq_tables* t, const tq_cache* c, const tq_diff_args* a,
                       bool precise, const RaggedAttend& rg, int hc, int pcta, const __half* qp,
                       int64_t qp_stride, int64_t grid, uint32_t* status, cudaStream_t st);
bool diff_attend_applies(const tq_geom* g, const tq_diff_args* a);
size_t diff_attend_workspace(const tq_geom* g, const tq_cache* c, const tq_diff_args* a);
int launch_diff_attend(const tq_geom* g, const tq_tables* t, const tq_cache* c, const tq_diff_args* a,
                       void* ws, uint32_t* status, cudaStream_t st);
// Whether some kernel attends a batch of this geometry, result type and engine.
bool attend_applies(const tq_geom* g, const tq_attend_args* a);
bool attend_few_applies(const tq_geom* g);
bool attend_mma_applies(const tq_geom* g);
int launch_attend_few(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                      const tq_attend_args* a, bool precise, const RaggedAttend& rg, int64_t Hkv,
                      int hc, int pcta, int rows, const __half* qp, int64_t qp_stride, int64_t grid,
                      uint32_t* status, cudaStream_t st);
int launch_attend_tc(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                     const tq_attend_args* a, const RaggedAttend& rg, int64_t Hkv, int64_t grid,
                     uint32_t* status, cudaStream_t st);
// fp16 and fp32 results ask for more than the fp16 operands that a bf16 one hides.
inline bool attend_precise(const tq_attend_args* a) { return a->out->dtype != TQ_BF16; }
int launch_attend_mma(const tq_geom* g, const tq_tables* t, const tq_cache* c,
                      const tq_attend_args* a, bool precise, const RaggedAttend& rg, int64_t Hkv,
                      int hc, int64_t grid, uint32_t* status, cudaStream_t st);

// cudaLaunchKernelEx with programmatic stream serialisation (see pdl_wait).
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                       cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}

}  // namespace tq
