// Host-side launchers of the state space block's kernels: selective scan, causal convolution, residual norm, 8-bit
// matrix product (internal to libsubq_b200).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.hpp"

namespace subq {

// [B, L, *] views with element strides (the innermost dimension contiguous); sg: between groups.
struct SelTensor {
    const void* p;
    int64_t sb, sl, sg;
    int vec;  // bytes that every row's start is a multiple of (16, 8, 4, 2)
};

struct SelParams {
    int B, L, D, N, G, Dg;  // Dg = D / G
    int softplus;
    SelTensor u, dt, z, Bm, C;  // z.p null: no gate
    SelTensor out;              // out.p null: not wanted
    const float* A;             // [D, N]
    const float* Dw;            // [D] or null
    const float* dt_bias;       // [D] or null
    const uint8_t* mask;
    int64_t mask_sb;
    const float* S_in;  // [B, D, N] or null
    float* S_out;       // or null
    // states before every kSelKeep-th token, [B, ceil(L / kSelKeep), D, 4 lanes] (lanes of a channel: sel_lanes(N)), or null
    float* kept;
    // segments of the sequence that are walked side by side
    int nseg, seg_tokens;  // tokens of a segment, a multiple of kSelTile
    float* seg_h;          // [nseg][B][D][4 lanes]: what a segment leaves of a zero state (backward: of a zero adjoint)
    float* seg_dt;         // [nseg][B][D]: sum of its step sizes
    // backward
    SelTensor dout, du, ddt, dz;
    void* dB; int64_t dB_sb, dB_sl, dB_sg;
    void* dC; int64_t dC_sb, dC_sl, dC_sg;
    const float* dS_out;  // gradient of the final state, or null
    float* dS_in;         // or null
    float* dA;            // [D, N]
    float* dD;            // [D] or null
    float* dbias;         // [D] or null
    // The walk back goes through every segment's tokens in ranges, from the last to the first, so that the parts of dB and dC
    // are of one range at a time.
    int range_tokens, range0;  // tokens of a range, a multiple of kSelTile; the begin of this launch's within a segment
    int rows;                  // tokens that part_bc has: L, or nseg * range_tokens
    float* carry;              // [nseg][B][D][4 lanes]: the adjoint between two ranges (null: one range)
    float* part_bc;            // [channel blocks of a group][B][rows][G][2][4 lanes]
    float* part_a;        // [B * nseg][D][4 lanes]
    float* part_d;        // [B * nseg][2][D]: dD, dbias
};
constexpr int kSelTile = 32;    // tokens that a CTA holds in shared memory
constexpr int kSelKeep = 8;     // tokens between two kept states
constexpr int kSelThreads = 256;
constexpr int kSelMaxN = 128;
constexpr int kSelResident = 4;  // CTAs of the walk that an SM holds (up to 32 states a channel; 2 above)
// Lanes of a channel, four states each.
inline int sel_lanes(int N) { return N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }
inline int sel_channels(int N) { return kSelThreads / sel_lanes(N); }  // channels of a CTA

enum SelPass { kSelSegments = 0, kSelWalk = 1 };
// One launch: the segments' states (kSelSegments: seg_h, seg_dt of all but the last) or the walk itself (out, kept, S_out).
cudaError_t launch_sel_fwd(const SelParams& p, int dtype, SelPass pass, cudaStream_t st);
// One launch: the segments' adjoints (of all but the first) or the walk back over a range with every gradient's part; then the
// sums of dB and dC of that range, and (`weights`, behind the last) of dA, dD and dbias.
cudaError_t launch_sel_bwd(const SelParams& p, int dtype, SelPass pass, cudaStream_t st);
cudaError_t launch_sel_sums(const SelParams& p, int dtype, bool weights, cudaStream_t st);
// Token by token without shared memory: single tokens and short calls.
cudaError_t launch_sel_step(const SelParams& p, int dtype, cudaStream_t st);

struct ConvParams {
    int B, L, D, W;
    int silu;
    SelTensor x, y;
    const float* w;     // [D, W]
    const float* bias;  // [D] or null
    const uint8_t* mask;
    int64_t mask_sb;
    const void* S_in;  // [B, W - 1, D] of x's type, or null
    void* S_out;       // or null; may be S_in
    // backward
    SelTensor dy, dx;
    const void* dS_out;  // or null
    void* dS_in;         // or null
    float* dw;           // [D, W]
    float* db;           // [D] or null
    float* part;         // [parts][W + 1][D]
    int parts, run;      // partial sums of a channel; groups of token runs of each
};
cudaError_t launch_conv_fwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches);
cudaError_t launch_conv_bwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches);
void conv_bwd_split(ConvParams& p);  // fills parts and run

struct RmsNormParams {
    int64_t rows;
    int D;
    float eps;
    const void* x; int64_t x_s;
    const void* res; int64_t res_s;  // or null
    void* r; int64_t r_s;            // x + res, or null
    void* y; int64_t y_s;
    float* scale; int64_t scale_s;   // y in 8 bits: one for every 128 columns
    const float* w;                  // or null (1)
    int norm;                        // 0: y is r itself (quantising alone)
    // backward (r is the input of the norm)
    const void* dy; int64_t dy_s;
    const void* dr; int64_t dr_s;    // gradient of r beside the norm's, or null
    void* dx; int64_t dx_s;          // of x's type
    void* dres; int64_t dres_s;      // of res's type, or null
    float* dw;                       // or null
    float* part;                     // [kRmsParts][D]
};
constexpr int kRmsMaxD = 16384;
constexpr int kRmsParts = 4 * 148;
// Types: x, r (res and r), y; y_dtype -1: e4m3 with scales.
cudaError_t launch_rms_norm(const RmsNormParams& p, int x_dtype, int r_dtype, int y_dtype, cudaStream_t st);
cudaError_t launch_rms_norm_bwd(const RmsNormParams& p, int x_dtype, int r_dtype, cudaStream_t st, int* launches);


// out[m, n] = bias[n] + sum over blocks kb of 128 of a_scale[m, kb] b_scale[n / 128, kb] (a[m, kb] . b[n, kb])
struct MatmulParams {
    int64_t M;
    int N, K, nk;                       // nk = ceil(K / 128)
    const void* a; int64_t a_s;         // e4m3, rows 16-byte aligned
    const void* b; int64_t b_s;
    const float* a_scale; int64_t as_s; // rows of nk
    const float* b_scale; int64_t bs_s;
    const float* bias;                  // or null
    void* out; int64_t out_s;
    int* status;
};
cudaError_t launch_scaled_matmul(const MatmulParams& p, int out_dtype, cudaStream_t st);

}  // namespace subq
