// Host-side launchers of the gated delta rule and layer norm kernels (internal to libsubq_b200).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.hpp"

namespace subq {

struct DeltaParams;

// Token-recurrent forward, any d, e <= 256 (delta_step.cu); S_out may be S_in.
cudaError_t launch_delta_step(const DeltaParams& p, int dtype, cudaStream_t st);
// Chunked forward, d <= 128 (delta_fwd.cuh): fills p.gates, p.Y and p.P, then walks the chunks. 2 launches, 4 with segments.
cudaError_t launch_delta_fwd_bf16(const DeltaParams& p, cudaStream_t st);
cudaError_t launch_delta_fwd_fp16(const DeltaParams& p, cudaStream_t st);
cudaError_t launch_delta_fwd_fp32(const DeltaParams& p, cudaStream_t st);
inline cudaError_t launch_delta_fwd(const DeltaParams& p, int dtype, cudaStream_t st) {
    return dtype == SUBQ_BF16 ? launch_delta_fwd_bf16(p, st) : dtype == SUBQ_FP16 ? launch_delta_fwd_fp16(p, st) : launch_delta_fwd_fp32(p, st);
}
// Gradients from what the forward left (p.gates, p.Y, p.P, p.S0, p.W) (delta_bwd.cuh). 2 launches, 4 with segments, and one per
// shared q, k, v.
cudaError_t launch_delta_bwd_bf16(const DeltaParams& p, cudaStream_t st, int* launches);
cudaError_t launch_delta_bwd_fp16(const DeltaParams& p, cudaStream_t st, int* launches);
cudaError_t launch_delta_bwd_fp32(const DeltaParams& p, cudaStream_t st, int* launches);
inline cudaError_t launch_delta_bwd(const DeltaParams& p, int dtype, cudaStream_t st, int* launches) {
    return dtype == SUBQ_BF16 ? launch_delta_bwd_bf16(p, st, launches)
                              : dtype == SUBQ_FP16 ? launch_delta_bwd_fp16(p, st, launches) : launch_delta_bwd_fp32(p, st, launches);
}

// Layer norm over the last dimension (layer_norm.cu): rows at element strides.
struct LnParams {
    int64_t rows;
    int D;
    float eps;
    const void* x; int64_t x_s;
    void* y; int64_t y_s;
    const void* dy; int64_t dy_s;
    void* dx; int64_t dx_s;
    const float* w;  // [D] or null (1)
    const float* b;  // [D] or null (0)
    float* dw;       // backward: [D] or null
    float* db;
    float* part;     // partial rows of (dw, db), or null (neither wanted)
    float* stats;    // D > 8192: mean and rsqrt of each row
};
constexpr int kLnPartials = 4 * 148;  // partial rows of (dw, db) at most
size_t ln_bwd_workspace_floats(int64_t rows, int D);
// The dtype pairs (x, y) are (T, T) for float32, float16, bfloat16 and (float32, float16 or bfloat16).
cudaError_t launch_layer_norm(const LnParams& p, int x_dtype, int y_dtype, bool bwd, cudaStream_t st, int* launches);

}  // namespace subq
