// Backward of the gated delta rule for float32 inputs (delta_bwd.cuh).
#include "delta_bwd.cuh"

namespace subq {

cudaError_t launch_delta_bwd_fp32(const DeltaParams& p, cudaStream_t st, int* launches) {
    return p.d <= 64 ? bwd_t<float, 64>(p, st, launches) : bwd_t<float, 128>(p, st, launches);
}

}  // namespace subq
