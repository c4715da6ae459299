// Token-recurrent gated delta rule: single-token decode steps, short calls, and
// heads above 128 dimensions. A CTA owns 32 value columns of one sequence and
// keeps S [d x 32] in the registers of its four warps: lane l of warp w has rows
// 16 i + 4 w + l / 8 and columns 4 (l % 8) .. + 3, so a row of the slice is one
// 128-byte access. S is read once and written once; per token
//   r = S^T k, s = S^T q (one reduction),  u = beta (v - gamma r),
//   S <- gamma S + k u^T,  o = scale (gamma s + (q.k) u),
// in float32. Bound by the state's 8 d e bytes for many sequences (one token),
// by launch latency for few.
#include "delta_common.cuh"
#include "delta_launch.h"
#include "scan_launch.h"

namespace subq {
namespace {

template <typename T, int RPL>
__global__ void __launch_bounds__(128) delta_step_kernel(const DeltaParams p, int vec) {
    __shared__ float red[2][4][32 * 2 + 4];  // [turn][warp][r | s of 32 columns, q.k]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ncb = (p.e + 31) / 32;
    const int64_t bh = blockIdx.x / ncb;
    const int b = (int)(bh / p.H), h = (int)(bh % p.H), col = (int)(blockIdx.x % ncb) * 32 + 4 * (lane & 7);
    const int row0 = 4 * warp + (lane >> 3);
    const T* k = static_cast<const T*>(p.k.p) + dl::tensor_base(p.k, b, h);
    const T* q = static_cast<const T*>(p.q.p) + dl::tensor_base(p.q, b, h);
    const T* v = static_cast<const T*>(p.v.p) + dl::tensor_base(p.v, b, h);
    T* o = static_cast<T*>(p.o.p) + dl::tensor_base(p.o, b, h);
    const float* S_in = p.S_in ? p.S_in + bh * p.d * p.e : nullptr;
    float S[RPL][4];
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
        const int row = 16 * i + row0;
        const float* src = S_in + (int64_t)row * p.e + col;
        if (S_in && row < p.d && vec && col < p.e) {
            const float4 x = *reinterpret_cast<const float4*>(src);
            S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = S_in && row < p.d && col + j < p.e ? src[j] : 0.f;
        }
    }
    int turn = 0;  // live tokens alternate between the two reduction buffers
    for (int n = 0; n < p.N; ++n) {
        if (p.mask && p.mask[(int64_t)b * p.mask_sb + n] == 0) {
            if (tid < 8)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < p.e) o[n * p.o.sn + col + j] = from_f<T>(0.f);
            continue;
        }
        float kr[RPL], sums[9] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const float gamma = p.lg.p ? expf(p.lg.p[b * p.lg.sb + h * p.lg.sh + n * p.lg.sn]) : 1.f;
        const float beta = p.beta.p ? p.beta.p[b * p.beta.sb + h * p.beta.sh + n * p.beta.sn] : 1.f;
        float vv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) vv[j] = col + j < p.e ? to_f<T>(v[n * p.v.sn + col + j]) : 0.f;
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
            const int row = 16 * i + row0;
            kr[i] = row < p.d ? to_f<T>(k[n * p.k.sn + row]) : 0.f;
            const float qr = row < p.d ? to_f<T>(q[n * p.q.sn + row]) : 0.f;
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
        for (int w = 0; w < 4; ++w) {
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
            for (int j = 0; j < 4; ++j) S[i][j] = fmaf(kr[i], u[j], gamma * S[i][j]);
        if (tid < 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < p.e) o[n * p.o.sn + col + j] = from_f<T>(p.scale * fmaf(qk, u[j], gamma * s[j]));
        turn ^= 1;
    }
    if (!p.S_out) return;
    float* S_out = p.S_out + bh * p.d * p.e;
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
        const int row = 16 * i + row0;
        if (row >= p.d) continue;
        float* dst = S_out + (int64_t)row * p.e + col;
        if (vec && col < p.e) {
            *reinterpret_cast<float4*>(dst) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < p.e) dst[j] = S[i][j];
        }
    }
}

template <typename T>
cudaError_t step_t(const DeltaParams& p, cudaStream_t st) {
    const unsigned blocks = (unsigned)((int64_t)p.B * p.H * ((p.e + 31) / 32));
    auto ok = [](const float* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
    const int vec = p.e % 4 == 0 && ok(p.S_in) && ok(p.S_out);
    if (p.d <= 32) delta_step_kernel<T, 2><<<blocks, 128, 0, st>>>(p, vec);
    else if (p.d <= 64) delta_step_kernel<T, 4><<<blocks, 128, 0, st>>>(p, vec);
    else if (p.d <= 128) delta_step_kernel<T, 8><<<blocks, 128, 0, st>>>(p, vec);
    else delta_step_kernel<T, 16><<<blocks, 128, 0, st>>>(p, vec);
    return cudaGetLastError();
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
