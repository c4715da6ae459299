// Selective scan kernels for float16 inputs.
#include "sel_bwd.cuh"

namespace subq {
cudaError_t launch_sel_fwd_fp16(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_fwd<__half>(p, pass, st); }
cudaError_t launch_sel_step_fp16(const SelParams& p, cudaStream_t st) { return sel::launch_step<__half>(p, st); }
cudaError_t launch_sel_bwd_fp16(const SelParams& p, SelPass pass, cudaStream_t st) { return sel::launch_bwd<__half>(p, pass, st); }
cudaError_t launch_sel_sums_fp16(const SelParams& p, bool weights, cudaStream_t st) { return sel::launch_sums<__half>(p, weights, st); }
}  // namespace subq
