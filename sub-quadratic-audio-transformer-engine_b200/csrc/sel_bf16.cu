// Selective scan kernels for bfloat16 inputs.
#include "sel_bwd.cuh"

namespace subq {
cudaError_t launch_sel_fwd_bf16(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_fwd<__nv_bfloat16>(p, pass, st); }
cudaError_t launch_sel_step_bf16(const SelParams& p, cudaStream_t st) { return sel::launch_step<__nv_bfloat16>(p, st); }
cudaError_t launch_sel_bwd_bf16(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_bwd<__nv_bfloat16>(p, pass, st); }
cudaError_t launch_sel_sums_bf16(const SelParams& p, bool weights, cudaStream_t st) { return sel::launch_sums<__nv_bfloat16>(p, weights, st); }
}  // namespace subq
