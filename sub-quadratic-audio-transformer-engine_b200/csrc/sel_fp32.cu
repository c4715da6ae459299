// Selective scan kernels for float32 inputs.
#include "sel_bwd.cuh"

namespace subq {
cudaError_t launch_sel_fwd_fp32(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_fwd<float>(p, pass, st); }
cudaError_t launch_sel_step_fp32(const SelParams& p, cudaStream_t st) { return sel::launch_step<float>(p, st); }
cudaError_t launch_sel_bwd_fp32(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_bwd<float>(p, pass, st); }
cudaError_t launch_sel_sums_fp32(const SelParams& p, bool weights, cudaStream_t st) { return sel::launch_sums<float>(p, weights, st); }
}  // namespace subq
