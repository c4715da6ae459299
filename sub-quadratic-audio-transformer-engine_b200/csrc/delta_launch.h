// Host-side launchers of the gated delta rule and layer norm kernels (internal to libsubq_b200).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace subq {

struct DeltaParams;

// Token-recurrent forward, any d, e <= 256 (delta_step.cu); S_out may be S_in.
cudaError_t launch_delta_step(const DeltaParams& p, int dtype, cudaStream_t st);
// Chunked forward, d <= 128 (delta_fwd.cu): fills p.Y, then walks the chunks. 2 launches.
cudaError_t launch_delta_fwd(const DeltaParams& p, int dtype, cudaStream_t st);
// Gradients from p.Y, p.S0 and p.W of the forward (delta_bwd.cu). 2 launches, and one per shared q, k, v.
cudaError_t launch_delta_bwd(const DeltaParams& p, int dtype, cudaStream_t st, int* launches);

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
constexpr int kLnLongSlices = 2 * 148;  // partial rows of the long-row form
size_t ln_bwd_workspace_floats(int64_t rows, int D);
// The dtype pairs (x, y) are (T, T) for float32, float16, bfloat16 and (float32, float16 or bfloat16).
cudaError_t launch_layer_norm(const LnParams& p, int x_dtype, int y_dtype, bool bwd, cudaStream_t st, int* launches);

}  // namespace subq
