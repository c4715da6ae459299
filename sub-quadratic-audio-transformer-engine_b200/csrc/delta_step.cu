// Token-recurrent gated delta rule: single-token decode steps, short calls, and
// heads above 128 dimensions. A tile is 32 value columns of one sequence;
// a CTA keeps S [d x 32] in the registers of its NW warps: lane l of warp w has
// rows 4 NW i + 4 w + l / 8 and columns 4 (l % 8) .. + 3, so a row of the slice is
// one 128-byte access. S is read once and written once; per token
//   r = S^T k, s = S^T q (one reduction),  u = beta (v - gamma r),
//   S <- gamma S + k u^T,  o = scale (gamma s + (q.k) u),
// in float32. Bound by the state's 8 d e bytes for many sequences (one token; 0.63
// of the measured copy bandwidth: the grid's second round is not full), by launch
// latency for few.
#include "delta_common.cuh"
#include "delta_launch.h"
#include "scan_launch.h"

namespace subq {
namespace {

// FULL: d is 4 NW RPL, e a multiple of 32 and the state aligned, so that no element needs a check.
template <typename T, int RPL, int NW, bool FULL>
__global__ void __launch_bounds__(32 * NW) delta_step_kernel(const DeltaParams p, int vec, unsigned tiles) {
    __shared__ float red[2][NW][32 * 2 + 4];  // [turn][warp][r | s of 32 columns, q.k]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ncb = (p.e + 31) / 32;
    const int row0 = 4 * warp + (lane >> 3);
    // (sequence, 32 columns) tiles; the next tile's state is on its way while one is computed
    float S[RPL][4], next[RPL][4];
    auto load = [&](unsigned tile) {
        const unsigned bh = tile / ncb;
        const int col = (int)(tile - bh * ncb) * 32 + 4 * (lane & 7);
        const float* S_in = p.S_in ? p.S_in + (int64_t)bh * p.d * p.e : nullptr;
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
            const int row = 4 * NW * i + row0;
            const float* src = S_in + (int64_t)row * p.e + col;
            if (S_in && (FULL || (row < p.d && vec && col < p.e))) {
                const float4 x = *reinterpret_cast<const float4*>(src);
                next[i][0] = x.x; next[i][1] = x.y; next[i][2] = x.z; next[i][3] = x.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) next[i][j] = !FULL && S_in && row < p.d && col + j < p.e ? src[j] : 0.f;
            }
        }
    };
    load(blockIdx.x);
    int turn = 0;  // live tokens alternate between the two reduction buffers
    for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const unsigned bh32 = tile / ncb;
        const int64_t bh = bh32;
        const int b = (int)(bh32 / (unsigned)p.H), h = (int)(bh32 - b * (unsigned)p.H), col = (int)(tile - bh32 * ncb) * 32 + 4 * (lane & 7);
        const T* k = static_cast<const T*>(p.k.p) + dl::tensor_base(p.k, b, h);
        const T* q = static_cast<const T*>(p.q.p) + dl::tensor_base(p.q, b, h);
        const T* v = static_cast<const T*>(p.v.p) + dl::tensor_base(p.v, b, h);
        T* o = static_cast<T*>(p.o.p) + dl::tensor_base(p.o, b, h);
#pragma unroll
        for (int i = 0; i < RPL; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = next[i][j];
        if (tile + gridDim.x < tiles) load(tile + gridDim.x);
        for (int n = 0; n < p.N; ++n) {
            if (p.mask && p.mask[(int64_t)b * p.mask_sb + n] == 0) {
                if (tid < 8)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (FULL || col + j < p.e) o[n * p.o.sn + col + j] = from_f<T>(0.f);
                continue;
            }
            float kr[RPL], sums[9] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            // The state's decay: gamma S, or S + (gamma - 1) S where gamma is near 1 (the series' rest is below 2^-26 of
            // S). Rounded by itself a gamma near 1 is off by up to 2^-25, the same way at every token (4096 tokens at
            // log gamma = -1e-4: the state 1.2e-4 off); and gamma - 1 has few bits of a small gamma.
            const float lg = p.lg.p ? p.lg.p[b * p.lg.sb + h * p.lg.sh + n * p.lg.sn] : 0.f, gamma = expf(lg);
            const bool near1 = fabsf(lg) < 0.0625f;
            const float decay = near1 ? lg * fmaf(lg, fmaf(lg, fmaf(lg, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f) : gamma;
            const float beta = p.beta.p ? p.beta.p[b * p.beta.sb + h * p.beta.sh + n * p.beta.sn] : 1.f;
            float vv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) vv[j] = FULL || col + j < p.e ? to_f<T>(v[n * p.v.sn + col + j]) : 0.f;
#pragma unroll
            for (int i = 0; i < RPL; ++i) {
                const int row = 4 * NW * i + row0;
                kr[i] = FULL || row < p.d ? to_f<T>(k[n * p.k.sn + row]) : 0.f;
                const float qr = FULL || row < p.d ? to_f<T>(q[n * p.q.sn + row]) : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sums[j] = fmaf(S[i][j], kr[i], sums[j]);
                    sums[4 + j] = fmaf(S[i][j], qr, sums[4 + j]);
                }
                sums[8] = fmaf(kr[i], qr, sums[8]);
            }
#pragma unroll
            for (int j = 0; j < 9; ++j) {
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 8);
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 16);
            }
            float(&mine)[68] = red[turn][warp];
            if (lane < 8) {
                *reinterpret_cast<float4*>(&mine[4 * lane]) = make_float4(sums[0], sums[1], sums[2], sums[3]);
                *reinterpret_cast<float4*>(&mine[32 + 4 * lane]) = make_float4(sums[4], sums[5], sums[6], sums[7]);
                if (lane == 0) mine[64] = sums[8];
            }
            __syncthreads();
            float r[4] = {0.f, 0.f, 0.f, 0.f}, s[4] = {0.f, 0.f, 0.f, 0.f}, qk = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float4 a = *reinterpret_cast<const float4*>(&red[turn][w][4 * (lane & 7)]);
                const float4 c = *reinterpret_cast<const float4*>(&red[turn][w][32 + 4 * (lane & 7)]);
                r[0] += a.x; r[1] += a.y; r[2] += a.z; r[3] += a.w;
                s[0] += c.x; s[1] += c.y; s[2] += c.z; s[3] += c.w;
                qk += red[turn][w][64];
            }
            float u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = beta * (vv[j] - gamma * r[j]);
#pragma unroll
            for (int i = 0; i < RPL; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) S[i][j] = fmaf(kr[i], u[j], fmaf(decay, S[i][j], near1 ? S[i][j] : 0.f));
            if (tid < 8)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (FULL || col + j < p.e) o[n * p.o.sn + col + j] = from_f<T>(p.scale * fmaf(qk, u[j], gamma * s[j]));
            turn ^= 1;
        }
        if (!p.S_out) continue;
        float* S_out = p.S_out + bh * p.d * p.e;
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
            const int row = 4 * NW * i + row0;
            if (!FULL && row >= p.d) continue;
            float* dst = S_out + (int64_t)row * p.e + col;
            if (FULL || (vec && col < p.e)) {
                *reinterpret_cast<float4*>(dst) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < p.e) dst[j] = S[i][j];
            }
        }
    }
}

template <typename T>
cudaError_t step_t(const DeltaParams& p, cudaStream_t st) {
    const unsigned tiles = (unsigned)((int64_t)p.B * p.H * ((p.e + 31) / 32));
    auto ok = [](const float* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
    const int vec = p.e % 4 == 0 && ok(p.S_in) && ok(p.S_out);
    auto run = [&](auto kernel, int threads, unsigned per_sm) {
        kernel<<<tiles < 148 * per_sm ? tiles : 148 * per_sm, threads, 0, st>>>(p, vec, tiles);
        return cudaGetLastError();
    };
    // two warps a tile: the work around a tile's 2048 state elements (d = 64) is as much as theirs, so fewer threads
    // with more elements each are faster (256 x 12 heads of 64 x 64: 24.6 us, 26.6 us with four warps). At 128 registers
    // 8 of the 10 CTAs an SM are resident (4 of 5 at d = 128): 1184 CTAs, then the other 296 on a quarter of the places.
    const bool full = vec && p.e % 32 == 0;
    if (p.d <= 32) return run(delta_step_kernel<T, 4, 2, false>, 64, 12);
    if (p.d == 64 && full) return run(delta_step_kernel<T, 8, 2, true>, 64, 10);
    if (p.d <= 64) return run(delta_step_kernel<T, 8, 2, false>, 64, 10);
    if (p.d == 128 && full) return run(delta_step_kernel<T, 16, 2, true>, 64, 5);
    if (p.d <= 128) return run(delta_step_kernel<T, 16, 2, false>, 64, 5);
    return run(delta_step_kernel<T, 16, 4, false>, 128, 2);
}

}  // namespace

cudaError_t launch_delta_step(const DeltaParams& p, int dtype, cudaStream_t st) {
    switch (dtype) {
        case SUBQ_FP32: return step_t<float>(p, st);
        case SUBQ_FP16: return step_t<__half>(p, st);
        case SUBQ_BF16: return step_t<__nv_bfloat16>(p, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace subq
