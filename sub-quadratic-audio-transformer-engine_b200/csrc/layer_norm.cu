// Layer norm over the last dimension of [rows, D], forward and backward:
//   xh = (x - mean(x)) rsqrt(var(x) + eps),   y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy
// with r the rsqrt (g is rounded to float32 the same way, by itself, wherever it is
// used, so that g - mean(g) is exactly 0 where it should be). Sums are float32 over
// values held in registers (the variance from the centred values); x, dy and y, dx
// have types of their own (a float32 residual stream normalised into bf16 and back
// is one pass each way).
//
// HBM-bound: a row is read once and written once. G threads hold a row, V
// consecutive elements (16 bytes of x) K times per thread; CTAs stay for many rows,
// with the next row on its way while one is worked on, so w and b are read once and
// the backward's dw and db stay in registers until the end: one partial row per CTA,
// summed by a second kernel in a fixed order (bitwise reproducible). Rows longer than
// the registers hold (D > 8192) are read again per pass, from L2.
// 65536 x 768, float32 -> bf16: forward 49 us (94 % of the measured copy bandwidth),
// backward 106 us (73 %: the registers that hold x, dy, dw and db leave room for two
// CTAs per SM, whose two sums a row are not hidden).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "delta_launch.h"
#include "kernels.hpp"
#include "scan_common.cuh"

namespace subq {
namespace {

constexpr int kThreads = 256;
constexpr int kSMs = 148;
constexpr int kPlainSmem = 40 * 1024;  // dynamic shared memory that a kernel has without asking (48 KB less what it declares)

// V elements as they are in memory: V of 16-byte pieces, of 8 bytes (4 of 16 bits) or single ones.
template <typename T, int V>
struct Raw {
    static constexpr int kBytes = V * (int)sizeof(T);
    using Piece = typename std::conditional<kBytes >= 16, uint4, typename std::conditional<kBytes == 8, uint2, T>::type>::type;
    static constexpr int kPieces = kBytes >= 16 ? kBytes / 16 : 1;
    Piece p[kPieces];
    __device__ __forceinline__ void load(const T* at) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) p[i] = reinterpret_cast<const Piece*>(at)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) p[i] = Piece{};
    }
    __device__ __forceinline__ void store(T* at) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) reinterpret_cast<Piece*>(at)[i] = p[i];
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
        const T* t = reinterpret_cast<const T*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f<T>(t[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
        T* t = reinterpret_cast<T*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from_f<T>(f[i]);
    }
};

// Sums of M values over the G threads of a row (G = 8, 32: lanes; 64, 128: warps of a part of the CTA; 256: the CTA).
template <int G, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float* red) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (G > 32) {
        const int group = threadIdx.x / G;
        auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(G) : "memory"); };
        sync();  // the sums of the call before have been read
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < M; ++i) red[(threadIdx.x >> 5) * M + i] = v[i];
        sync();
#pragma unroll
        for (int i = 0; i < M; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < G / 32; ++w) v[i] += red[(group * (G / 32) + w) * M + i];
        }
    }
}

template <typename TX, typename TY, int G, int V, int K>
__global__ void __launch_bounds__(kThreads, K * V <= 16 ? 3 : K * V <= 24 ? 2 : 1) ln_fwd_kernel(const LnParams p) {
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
    Raw<TX, V> next[K];  // the next row, on its way
    auto load = [&](int64_t row) {
        const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (row < p.rows && c < D) next[k].load(x + c);
            else next[k].zero();
        }
    };
    const int64_t first = (int64_t)blockIdx.x * kRows;
    load(first + threadIdx.x / G);
    // the loop runs the same number of times in every thread of a row's group and of a warp
#pragma unroll 1
    for (int64_t r0 = first; r0 < p.rows; r0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = r0 + threadIdx.x / G;
        float f[K][V], s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) next[k].get(f[k]);
        if (r0 + (int64_t)gridDim.x * kRows < p.rows) load(row + (int64_t)gridDim.x * kRows);
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
            if (row < p.rows && c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) f[k][i] = fmaf(f[k][i] * r, w[k][i], b[k][i]);
                Raw<TY, V> out;
                out.set(f[k]);
                out.store(y + c);
            }
        }
    }
}

// CTAs per SM that the backward's registers are cut for (8 single elements: two rows of them on their way, 64 registers
// spill; width 511: 65 us, 100 with four CTAs; 2047: 71 us with two, 93 with three).
constexpr int bwd_ctas(int G, int V, int K) {
    if (V == 1 && K == 8) return G == kThreads ? 2 : 3;
    return K * V <= 8 ? 4 : K * V <= 24 ? 2 : 1;
}

// N bytes (8 or 16) straight to shared memory.
template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(src), "n"(N) : "memory");
}

// Bytes of shared memory in which a thread's pieces of the next row wait, where the registers do not hold them. With
// float32 x or up to 16 elements a thread (backward, 49152 x 1024 float32: 118 us without, 99 us with; 65536 x 768 bf16,
// 24 elements: 84 us without, 95 us with).
template <typename TX, typename TY, int V, int K>
constexpr int stage_bytes() {
    return V > 1 && K * V > 8 && (V == 4 || K * V <= 16) ? kThreads * K * V * (int)(sizeof(TX) + sizeof(TY)) : 0;
}

template <typename TX, typename TY, int G, int V, int K>
__global__ void __launch_bounds__(kThreads, bwd_ctas(G, V, K)) ln_bwd_kernel(const LnParams p) {
    __shared__ float red[kThreads / 32 * 2];
    // stage, [D] weight, [D] sums of the rows a CTA handles side by side
    extern __shared__ __align__(16) unsigned char raw_ln[];
    float* sm_ln = reinterpret_cast<float*>(raw_ln + stage_bytes<TX, TY, V, K>());
    float* cols = sm_ln + p.D;
    constexpr int kRows = kThreads / G;
    const int li = threadIdx.x % G, D = p.D;
    const float inv = 1.f / D;
    for (int c = threadIdx.x; c < D; c += kThreads) sm_ln[c] = p.w ? p.w[c] : 1.f;
    __syncthreads();
    float dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
    // The next row of x and dy is on its way while one is worked on: in registers up to 8 elements a thread, else in
    // slots of shared memory that each thread fills and empties for itself, else not (see stage_bytes).
    constexpr bool kAhead = K * V <= 8, kStage = stage_bytes<TX, TY, V, K>() > 0;
    constexpr int kBx = 16, kBy = V > 1 ? V * (int)sizeof(TY) : 16;  // bytes of a piece of x (V > 1) and of dy
    constexpr int kPy = kBy > 16 ? kBy / 16 : 1, kBp = kBy / kPy;
    unsigned char* slot_x = raw_ln + threadIdx.x * kBx;                         // [K][thread]
    unsigned char* slot_y = raw_ln + kThreads * K * kBx + threadIdx.x * kBp;    // [K][piece][thread]
    auto send = [&](int64_t row) {
        if (row < p.rows) {
            const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
            const TY* dy = static_cast<const TY*>(p.dy) + row * p.dy_s;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * G + li) * V;
                if (c < D) {
                    copy_async<kBx>(slot_x + k * kThreads * kBx, x + c);
#pragma unroll
                    for (int i = 0; i < kPy; ++i)
                        copy_async<kBp>(slot_y + (k * kPy + i) * kThreads * kBp, reinterpret_cast<const unsigned char*>(dy + c) + i * kBp);
                }
            }
        }
    };
    Raw<TX, V> nx[K];
    Raw<TY, V> ny[K];
    auto load = [&](int64_t row) {
        const TX* x = static_cast<const TX*>(p.x) + row * p.x_s;
        const TY* dy = static_cast<const TY*>(p.dy) + row * p.dy_s;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (row < p.rows && c < D) {
                nx[k].load(x + c);
                ny[k].load(dy + c);
            } else {
                nx[k].zero();
                ny[k].zero();
            }
        }
    };
    const int64_t first = (int64_t)blockIdx.x * kRows;
    if (kAhead) load(first + threadIdx.x / G);
    if constexpr (kStage) send(first + threadIdx.x / G);
#pragma unroll 1
    for (int64_t r0 = first; r0 < p.rows; r0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = r0 + threadIdx.x / G;
        float f[K][V], e[K][V], s[2] = {0.f, 0.f};
        if constexpr (kStage) {
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const bool in = row < p.rows && (k * G + li) * V < D;
                nx[k].zero();
                ny[k].zero();
                if (in) {
                    nx[k].p[0] = *reinterpret_cast<const typename Raw<TX, V>::Piece*>(slot_x + k * kThreads * kBx);
#pragma unroll
                    for (int i = 0; i < kPy; ++i)
                        ny[k].p[i] = *reinterpret_cast<const typename Raw<TY, V>::Piece*>(slot_y + (k * kPy + i) * kThreads * kBp);
                }
            }
        } else if (!kAhead) {
            load(row);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            nx[k].get(f[k]);
            ny[k].get(e[k]);
        }
        if (kAhead && r0 + (int64_t)gridDim.x * kRows < p.rows) load(row + (int64_t)gridDim.x * kRows);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (c < D)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[0] += f[k][i];
                    s[1] += __fmul_rn(e[k][i], sm_ln[c + i]);
                }
        }
        row_sums<G, 2>(s, red);
        // (the sums have taken every slot's values: the slots are free)
        if constexpr (kStage) send(row + (int64_t)gridDim.x * kRows);
        const float mean = s[0] * inv, mg = s[1] * inv;
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (c < D)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    f[k][i] -= mean;
                    s[0] = fmaf(f[k][i], f[k][i], s[0]);
                    s[1] = fmaf(e[k][i] * sm_ln[c + i], f[k][i], s[1]);
                }
        }
        row_sums<G, 2>(s, red);
        const float r = rsqrtf(s[0] * inv + p.eps), mgx = s[1] * inv * r;
        TX* dx = static_cast<TX*>(p.dx) + row * p.dx_s;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + li) * V;
            if (row < p.rows && c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = f[k][i] * r;
                    dw[k][i] = fmaf(e[k][i], xh, dw[k][i]);
                    db[k][i] += e[k][i];
                    f[k][i] = r * (__fmul_rn(e[k][i], sm_ln[c + i]) - mg - xh * mgx);
                }
                Raw<TX, V> out;
                out.set(f[k]);
                out.store(dx + c);
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

// dw[c], db[c]: the nb partial rows added by 32 threads a column, each every 32nd row in order, then those in order.
__global__ void __launch_bounds__(1024) ln_cols_kernel(const float* part, int nb, int D, float* dw, float* db) {
    __shared__ float red[32][33];
    const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float s = 0.f;
    if (c < D)
#pragma unroll 4
        for (int i = k; i < nb; i += 32) s += part[((int64_t)i * 2 + which) * D + c];
    red[k][threadIdx.x & 31] = s;
    __syncthreads();
    float* out = which ? db : dw;
    if (k == 0 && c < D && out) {
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][threadIdx.x];
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

// Threads per row and elements per thread: the smallest group of threads that hold at most `most` elements of the row
// each, V of them (16 bytes of x) at a time where every row of x, y and their gradients starts on a 16-byte boundary and
// the width allows it, single ones otherwise. G = 0: the row is too long.
//
// Fewer threads a row are more rows in flight per SM and shorter sums, until the registers run out. Measured, us, about
// 50 M elements (25 M at the odd widths), the threads taken first, then the next choice:
//   forward, float32 -> bf16   width 64: 8 10, 32 14;  256: 32 23, 8 27;  768: 32 55, 64 57;  1280: 64 57, 32 70;  2048: 128 55, 256 59
//   backward, float32, bf16    width 64: 32 33, 8 49;  512: 32 79, 64 91;  1024: 64 99, 128 116;  1280: 64 114, 128 116 (bf16: 93, 106)
//   forward, odd widths        511: 32 39, 64 43;  767: 64 43, 32 53;  2047: 128 37, 256 43
//   backward, odd widths       129: 32 42, 64 50;  511: 64 65, 128 75;  1021: 128 69, 64 77, 256 85;  2047: 256 71, 128 75
Shape shape_of(int D, bool vec, int V, bool bwd) {
    if (!vec || D % V != 0) V = 1;
    const int n = D / V, most = V > 1 ? 24 : bwd ? 8 : 16;
    auto each = [&](int G) { return (n + G - 1) / G; };
    int G = V > 1 && !bwd ? 8 : 32;
    while (G < kThreads && each(G) * V > most) G = G == 8 ? 32 : 2 * G;
    const int k = each(G);
    if (k * V > 32) return {0, 1, 0};
    return {G, V, V > 1 ? k : k <= 4 ? 4 : k <= 8 ? 8 : k <= 16 ? 16 : 32};
}

template <typename F>
int resident(F kernel, size_t smem) {
    int n = 0;
    if ((smem > kPlainSmem && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, smem) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = 1;
    }
    return n;
}

bool vec_of(const LnParams& p, bool bwd, int dx_size, int dy_size) {
    auto ok = [](const void* q, int64_t s, int size) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (s * size) % 16 == 0; };
    if (!ok(p.x, p.x_s, dx_size)) return false;
    return bwd ? ok(p.dy, p.dy_s, dy_size) && ok(p.dx, p.dx_s, dx_size) : ok(p.y, p.y_s, dy_size);
}

// Launches as many CTAs as fit at once (the backward at most kLnPartials: a partial row each), or fewer.
template <typename TX, typename TY, int G, int V, int K>
cudaError_t run(const LnParams& p, bool bwd, int* blocks, cudaStream_t st) {
    constexpr int64_t kRows = kThreads / G;
    const int64_t need = (p.rows + kRows - 1) / kRows;
    if (!bwd) {
        static const int per_sm = resident(ln_fwd_kernel<TX, TY, G, V, K>, 0);
        *blocks = (int)(need < kSMs * per_sm ? need : kSMs * per_sm);
        ln_fwd_kernel<TX, TY, G, V, K><<<*blocks, kThreads, 0, st>>>(p);
    } else if constexpr (G > 8 && (V > 1 || K <= 8 || G == kThreads)) {
        constexpr int kStage = stage_bytes<TX, TY, V, K>();
        constexpr int kMost = kStage + (G < kThreads ? 2 : 1) * (int)sizeof(float) * G * V * K;  // of the widest row
        const int smem = kStage + p.D * (p.part && G < kThreads ? 2 : 1) * (int)sizeof(float);
        static const int per_sm = resident(ln_bwd_kernel<TX, TY, G, V, K>, kMost);
        const int64_t most = kSMs * per_sm < kLnPartials ? kSMs * per_sm : kLnPartials;
        *blocks = (int)(need < most ? need : most);
        if (smem > kPlainSmem) {  // (every call sets the same limit: calls from other threads, of other widths, may be between here and the launch)
            const cudaError_t err = cudaFuncSetAttribute(ln_bwd_kernel<TX, TY, G, V, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
            if (err != cudaSuccess) return err;
        }
        ln_bwd_kernel<TX, TY, G, V, K><<<*blocks, kThreads, smem, st>>>(p);
    } else {
        return cudaErrorInvalidValue;  // (shape_of gives the backward no such shape)
    }
    return cudaGetLastError();
}

template <typename TX, typename TY, int G>
cudaError_t run_g(const LnParams& p, const Shape& s, bool bwd, int* blocks, cudaStream_t st) {
    constexpr int V = 16 / sizeof(TX);
    constexpr bool kAll = G == kThreads;  // (up to 32 elements a thread, see shape_of)
    if (s.V == V) switch (s.K) {
        case 1: return run<TX, TY, G, V, 1>(p, bwd, blocks, st);
        case 2: return run<TX, TY, G, V, 2>(p, bwd, blocks, st);
        case 3: return run<TX, TY, G, V, 3>(p, bwd, blocks, st);
        default:
            if constexpr (V == 4) {
                if (s.K == 4) return run<TX, TY, G, V, 4>(p, bwd, blocks, st);
                if (s.K <= 6) return run<TX, TY, G, V, 6>(p, bwd, blocks, st);
            }
            if constexpr (kAll) return run<TX, TY, G, V, 32 / V>(p, bwd, blocks, st);
    }
    if constexpr (G > 8) switch (s.K) {
        case 4: return run<TX, TY, G, 1, 4>(p, bwd, blocks, st);
        case 8: return run<TX, TY, G, 1, 8>(p, bwd, blocks, st);
        case 16: return run<TX, TY, G, 1, 16>(p, bwd, blocks, st);
        default:
            if constexpr (kAll) return run<TX, TY, G, 1, 32>(p, bwd, blocks, st);
    }
    return cudaErrorInvalidValue;
}

template <typename TX, typename TY>
cudaError_t ln_t(LnParams p, bool bwd, cudaStream_t st, int* launches) {
    const Shape s = shape_of(p.D, vec_of(p, bwd, sizeof(TX), sizeof(TY)), 16 / sizeof(TX), bwd);
    *launches = 1;
    cudaError_t err;
    int partial_rows = 1;
    if (s.G == 8) {
        err = run_g<TX, TY, 8>(p, s, bwd, &partial_rows, st);
    } else if (s.G == 32) {
        err = run_g<TX, TY, 32>(p, s, bwd, &partial_rows, st);
    } else if (s.G == 64) {
        err = run_g<TX, TY, 64>(p, s, bwd, &partial_rows, st);
    } else if (s.G == 128) {
        err = run_g<TX, TY, 128>(p, s, bwd, &partial_rows, st);
    } else if (s.G) {
        err = run_g<TX, TY, kThreads>(p, s, bwd, &partial_rows, st);
    } else {
        const int64_t most = kSMs * 8;
        const unsigned grid = (unsigned)(p.rows < most ? p.rows : most);
        if (bwd) ln_long_kernel<TX, TY, true><<<grid, kThreads, 0, st>>>(p);
        else ln_long_kernel<TX, TY, false><<<grid, kThreads, 0, st>>>(p);
        err = cudaGetLastError();
        if (err == cudaSuccess && p.part) {
            partial_rows = (int)(p.rows < kLnPartials ? p.rows : kLnPartials);
            ln_long_cols_kernel<TX, TY><<<dim3((p.D + kThreads - 1) / kThreads, partial_rows), kThreads, 0, st>>>(p);
            err = cudaGetLastError();
            ++*launches;
        }
    }
    if (err == cudaSuccess && p.part) {
        ln_cols_kernel<<<dim3((p.D + 31) / 32, 2), 1024, 0, st>>>(p.part, partial_rows, p.D, p.dw, p.db);
        err = cudaGetLastError();
        ++*launches;
    }
    return err;
}

}  // namespace

// Partial rows of (dw, db), and for long rows each row's mean and rsqrt.
size_t ln_bwd_workspace_floats(int64_t rows, int D) {
    const int64_t most = kLnPartials;
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
