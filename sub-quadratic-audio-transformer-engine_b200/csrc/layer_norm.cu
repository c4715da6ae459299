// Layer norm over the last dimension of [rows, D], forward and backward:
//   xh = (x - mean(x)) rsqrt(var(x) + eps),   y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy
// with r the rsqrt (g is rounded to float32 the same way, by itself, wherever it
// is used, so that g - mean(g) is exactly 0 where it should be). Sums are float32 over values held in registers (the variance
// from the centred values); x, dy and y, dx have types of their own (a float32
// residual stream normalised into bf16 and back is one pass each way).
//
// HBM-bound: a row is read once and written once. kG threads hold a row, V
// consecutive elements (16 or 32 bytes) K times per thread; CTAs stay for many
// rows, so w and b are read once per thread and the backward's dw and db stay in
// registers until the end: one partial row per CTA, summed by a second kernel in
// a fixed order (bitwise reproducible). Rows longer than the registers hold
// (D > 8192) are read again per pass, from L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "delta_launch.h"
#include "kernels.hpp"
#include "scan_common.cuh"

namespace subq {
namespace {

constexpr int kThreads = 256;
constexpr int kSMs = 148;

template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&f)[V]) {
    if constexpr (V == 1) {
        f[0] = to_f<T>(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            T t[2];
            *reinterpret_cast<uint32_t*>(t) = w[i];
            f[2 * i] = to_f<T>(t[0]);
            f[2 * i + 1] = to_f<T>(t[1]);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&f)[V]) {
    if constexpr (V == 1) {
        *p = from_f<T>(f[0]);
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        alignas(16) T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = from_f<T>(f[i]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
    }
}

// Sums of M values over the G threads of a row (G = 8, 32: lanes; 256: the CTA).
template <int G, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float* red) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (G == kThreads) {
        __syncthreads();  // the sums of the call before have been read
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < M; ++i) red[(threadIdx.x >> 5) * M + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < M; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w) v[i] += red[w * M + i];
        }
    }
}

template <typename TX, typename TY, int G, int V, int K>
__global__ void __launch_bounds__(kThreads) ln_fwd_kernel(const LnParams p) {
    __shared__ float red[kThreads / 32];
    constexpr int kRows = kThreads / G;
    const int li = threadIdx.x % G, D = p.D;
    const float inv = 1.f / D;
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (k * G + li) * V + i;
            w[k][i] = p.w && c < D ? p.w[c] : 1.f;
            b[k][i] = p.b && c < D ? p.b[c] : 0.f;
        }
    // the loop runs the same number of times in every thread of a row's group and of a warp
#pragma unroll 1
    for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < p.rows; r0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = r0 + threadIdx.x / G;
        const bool live = row < p.rows;
        const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
        float f[K][V], s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (live && c < D) load_v<TX, V>(x + c, f[k]);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) f[k][i] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += f[k][i];
        row_sums<G, 1>(s, red);
        const float mean = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if ((k * G + li) * V < D)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    f[k][i] -= mean;
                    s[0] = fmaf(f[k][i], f[k][i], s[0]);
                }
        row_sums<G, 1>(s, red);
        const float r = rsqrtf(s[0] * inv + p.eps);
        TY* y = static_cast<TY*>(p.y) + row * p.y_s;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (live && c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) f[k][i] = fmaf(f[k][i] * r, w[k][i], b[k][i]);
                store_v<TY, V>(y + c, f[k]);
            }
        }
    }
}

template <typename TX, typename TY, int G, int V, int K>
__global__ void __launch_bounds__(kThreads) ln_bwd_kernel(const LnParams p) {
    __shared__ float red[kThreads / 32 * 2];
    extern __shared__ float cols[];  // [D] sums of the rows a CTA handles side by side
    constexpr int kRows = kThreads / G;
    const int li = threadIdx.x % G, D = p.D;
    const float inv = 1.f / D;
    float w[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (k * G + li) * V + i;
            w[k][i] = p.w && c < D ? p.w[c] : 1.f;
            dw[k][i] = db[k][i] = 0.f;
        }
#pragma unroll 1
    for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < p.rows; r0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = r0 + threadIdx.x / G;
        const bool live = row < p.rows;
        const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
        const TY* dy = static_cast<const TY*>(p.dy) + row * p.dy_s;
        float f[K][V], e[K][V], s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (live && c < D) {
                load_v<TX, V>(x + c, f[k]);
                load_v<TY, V>(dy + c, e[k]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) f[k][i] = e[k][i] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[0] += f[k][i];
                s[1] += __fmul_rn(e[k][i], w[k][i]);
            }
        row_sums<G, 2>(s, red);
        const float mean = s[0] * inv, mg = s[1] * inv;
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if ((k * G + li) * V < D)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    f[k][i] -= mean;
                    s[0] = fmaf(f[k][i], f[k][i], s[0]);
                    s[1] = fmaf(e[k][i] * w[k][i], f[k][i], s[1]);
                }
        row_sums<G, 2>(s, red);
        const float r = rsqrtf(s[0] * inv + p.eps), mgx = s[1] * inv * r;
        TX* dx = static_cast<TX*>(p.dx) + row * p.dx_s;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (live && c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = f[k][i] * r;
                    dw[k][i] = fmaf(e[k][i], xh, dw[k][i]);
                    db[k][i] += e[k][i];
                    f[k][i] = r * (__fmul_rn(e[k][i], w[k][i]) - mg - xh * mgx);
                }
                store_v<TX, V>(dx + c, f[k]);
            }
        }
    }
    if (!p.part) return;
    // this CTA's row of partial sums, its row slots added in order
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* part = p.part + ((int64_t)blockIdx.x * 2 + which) * D;
        for (int slot = 0; slot < kRows; ++slot) {
            if (threadIdx.x / G == slot)
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int c = (k * G + li) * V + i;
                        const float v = which ? db[k][i] : dw[k][i];
                        if (c < D) {
                            const float sum = slot ? cols[c] + v : v;
                            if (slot == kRows - 1) part[c] = sum;
                            else cols[c] = sum;
                        }
                    }
            __syncthreads();
        }
    }
}

// dw[c], db[c]: the nb partial rows added in order by 8 threads a column, then those in order.
__global__ void __launch_bounds__(256) ln_cols_kernel(const float* part, int nb, int D, float* dw, float* db) {
    __shared__ float red[8][33];
    const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float s = 0.f;
    if (c < D)
#pragma unroll 8
        for (int i = k; i < nb; i += 8) s += part[((int64_t)i * 2 + which) * D + c];
    red[k][threadIdx.x & 31] = s;
    __syncthreads();
    float* out = which ? db : dw;
    if (k == 0 && c < D && out) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
        out[c] = s;
    }
}

// ---- rows of any length: a CTA per row, the row read again for each pass
template <typename TX, typename TY, bool BWD>
__global__ void __launch_bounds__(kThreads) ln_long_kernel(const LnParams p) {
    __shared__ float red[kThreads / 32 * 2];
    const int D = p.D;
    const float inv = 1.f / D;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
        const TY* dy = BWD ? static_cast<const TY*>(p.dy) + row * p.dy_s : nullptr;
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < D; c += kThreads) {
            s[0] += to_f<TX>(x[c]);
            if (BWD) s[1] += __fmul_rn(to_f<TY>(dy[c]), p.w ? p.w[c] : 1.f);
        }
        row_sums<kThreads, 2>(s, red);
        const float mean = s[0] * inv, mg = s[1] * inv;
        s[0] = s[1] = 0.f;
        for (int c = threadIdx.x; c < D; c += kThreads) {
            const float v = to_f<TX>(x[c]) - mean;
            s[0] = fmaf(v, v, s[0]);
            if (BWD) s[1] = fmaf(to_f<TY>(dy[c]) * (p.w ? p.w[c] : 1.f), v, s[1]);
        }
        row_sums<kThreads, 2>(s, red);
        const float r = rsqrtf(s[0] * inv + p.eps), mgx = s[1] * inv * r;
        if (BWD && p.stats && threadIdx.x == 0) {
            p.stats[2 * row] = mean;
            p.stats[2 * row + 1] = r;
        }
        for (int c = threadIdx.x; c < D; c += kThreads) {
            const float xh = (to_f<TX>(x[c]) - mean) * r, w = p.w ? p.w[c] : 1.f;
            if (BWD) static_cast<TX*>(p.dx)[row * p.dx_s + c] = from_f<TX>(r * (__fmul_rn(to_f<TY>(dy[c]), w) - mg - xh * mgx));
            else static_cast<TY*>(p.y)[row * p.y_s + c] = from_f<TY>(fmaf(xh, w, p.b ? p.b[c] : 0.f));
        }
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kThreads) ln_long_cols_kernel(const LnParams p) {  // a column per thread, a slice of rows per blockIdx.y
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= p.D) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float e = to_f<TY>(static_cast<const TY*>(p.dy)[row * p.dy_s + c]);
        const float xh = (to_f<TX>(static_cast<const TX*>(p.x)[row * p.x_s + c]) - p.stats[2 * row]) * p.stats[2 * row + 1];
        dw = fmaf(e, xh, dw);
        db += e;
    }
    p.part[((int64_t)blockIdx.y * 2) * p.D + c] = dw;
    p.part[((int64_t)blockIdx.y * 2 + 1) * p.D + c] = db;
}

struct Shape {
    int G, V, K;
};

// Threads per row and elements per thread: the smallest group whose threads hold
// at most 32 elements each; 8 elements at a time where every row starts on a
// 16-byte boundary, single ones otherwise. G = 0: the row is too long.
Shape shape_of(int D, bool vec) {
    if (vec && D % 8 == 0) {
        const int n = D / 8;
        if (n <= 32) return {8, 8, (n + 7) / 8};
        if (n <= 128) return {32, 8, (n + 31) / 32};
        if (n <= 1024) return {kThreads, 8, (n + kThreads - 1) / kThreads};
        return {0, 1, 0};
    }
    const int G = D <= 1024 ? 32 : kThreads;
    const int k = (D + G - 1) / G;
    if (k > 32) return {0, 1, 0};
    return {G, 1, k <= 8 ? 8 : k <= 16 ? 16 : 32};
}

bool vec_of(const LnParams& p, bool bwd, int dx_size, int dy_size) {
    auto ok = [](const void* q, int64_t s, int size) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (s * size) % 16 == 0; };
    if (!ok(p.x, p.x_s, dx_size)) return false;
    return bwd ? ok(p.dy, p.dy_s, dy_size) && ok(p.dx, p.dx_s, dx_size) : ok(p.y, p.y_s, dy_size);
}

template <typename TX, typename TY, int G, int V, int K>
cudaError_t run(const LnParams& p, bool bwd, int blocks, cudaStream_t st) {
    if (bwd) ln_bwd_kernel<TX, TY, G, V, K><<<blocks, kThreads, p.part && G < kThreads ? p.D * sizeof(float) : 0, st>>>(p);
    else ln_fwd_kernel<TX, TY, G, V, K><<<blocks, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename TX, typename TY, int G>
cudaError_t run_g(const LnParams& p, const Shape& s, bool bwd, int blocks, cudaStream_t st) {
    if (s.V == 8) switch (s.K) {
        case 1: return run<TX, TY, G, 8, 1>(p, bwd, blocks, st);
        case 2: return run<TX, TY, G, 8, 2>(p, bwd, blocks, st);
        case 3: return run<TX, TY, G, 8, 3>(p, bwd, blocks, st);
        default: return run<TX, TY, G, 8, 4>(p, bwd, blocks, st);
    }
    if constexpr (G > 8) switch (s.K) {
        case 8: return run<TX, TY, G, 1, 8>(p, bwd, blocks, st);
        case 16: return run<TX, TY, G, 1, 16>(p, bwd, blocks, st);
        default: return run<TX, TY, G, 1, 32>(p, bwd, blocks, st);
    }
    return cudaErrorInvalidValue;
}

int blocks_of(const LnParams& p, const Shape& s, bool bwd) {
    const int64_t rows = s.G ? kThreads / s.G : 1, need = (p.rows + rows - 1) / rows;
    // 2 CTAs per SM fit with the backward's sums in registers; the forward's 8
    const int64_t most = kSMs * (bwd ? 2 : 8);
    return (int)(need < most ? (need > 0 ? need : 1) : most);
}

template <typename TX, typename TY>
cudaError_t ln_t(LnParams p, bool bwd, cudaStream_t st, int* launches) {
    const Shape s = shape_of(p.D, vec_of(p, bwd, sizeof(TX), sizeof(TY)));
    const int blocks = blocks_of(p, s, bwd);
    *launches = 1;
    cudaError_t err;
    int partial_rows = blocks;
    if (s.G == 8) {
        err = run_g<TX, TY, 8>(p, s, bwd, blocks, st);
    } else if (s.G == 32) {
        err = run_g<TX, TY, 32>(p, s, bwd, blocks, st);
    } else if (s.G) {
        err = run_g<TX, TY, kThreads>(p, s, bwd, blocks, st);
    } else {
        const int64_t most = kSMs * 8;
        const unsigned grid = (unsigned)(p.rows < most ? p.rows : most);
        if (bwd) ln_long_kernel<TX, TY, true><<<grid, kThreads, 0, st>>>(p);
        else ln_long_kernel<TX, TY, false><<<grid, kThreads, 0, st>>>(p);
        err = cudaGetLastError();
        if (err == cudaSuccess && p.part) {
            partial_rows = (int)(p.rows < kLnLongSlices ? p.rows : kLnLongSlices);
            ln_long_cols_kernel<TX, TY><<<dim3((p.D + kThreads - 1) / kThreads, partial_rows), kThreads, 0, st>>>(p);
            err = cudaGetLastError();
            ++*launches;
        }
    }
    if (err == cudaSuccess && p.part) {
        ln_cols_kernel<<<dim3((p.D + 31) / 32, 2), 256, 0, st>>>(p.part, partial_rows, p.D, p.dw, p.db);
        err = cudaGetLastError();
        ++*launches;
    }
    return err;
}

}  // namespace

// Partial rows of (dw, db), and for long rows each row's mean and rsqrt.
size_t ln_bwd_workspace_floats(int64_t rows, int D) {
    const int64_t most = kSMs * 2;
    return (size_t)2 * D * (rows < most ? rows : most) + (D > 8192 ? (size_t)2 * rows : 0);
}

cudaError_t launch_layer_norm(const LnParams& p, int x_dtype, int y_dtype, bool bwd, cudaStream_t st, int* launches) {
    if (x_dtype == SUBQ_FP32 && y_dtype == SUBQ_FP32) return ln_t<float, float>(p, bwd, st, launches);
    if (x_dtype == SUBQ_FP32 && y_dtype == SUBQ_BF16) return ln_t<float, __nv_bfloat16>(p, bwd, st, launches);
    if (x_dtype == SUBQ_FP32 && y_dtype == SUBQ_FP16) return ln_t<float, __half>(p, bwd, st, launches);
    if (x_dtype == SUBQ_BF16 && y_dtype == SUBQ_BF16) return ln_t<__nv_bfloat16, __nv_bfloat16>(p, bwd, st, launches);
    if (x_dtype == SUBQ_FP16 && y_dtype == SUBQ_FP16) return ln_t<__half, __half>(p, bwd, st, launches);
    return cudaErrorInvalidValue;
}

}  // namespace subq
