// Chunked forward of the gated delta rule for float16 inputs (delta_fwd.cuh; one
// translation unit per type, so that they compile side by side).
#include "delta_fwd.cuh"

namespace subq {

cudaError_t launch_delta_fwd_fp16(const DeltaParams& p, cudaStream_t st) {
    return p.d <= 64 ? fwd_t<__half, 64>(p, st) : fwd_t<__half, 128>(p, st);
}

}  // namespace subq
