// Short causal convolution over [B, L, D], one filter of W = 2, 3 or 4 taps a channel, forward and backward:
//   pre_t = b + sum_j w_j x_{t-W+1+j},   y_t = silu(pre_t) or pre_t.
// Before the first token stands the carried window (the W - 1 inputs before it, zeros without one); a masked token's input
// counts as 0 and its output is 0; the window that is handed on is of the W - 1 inputs up to the last live token.
//   dpre_t = dy_t act'(pre_t),   dx_s = sum_j w_j dpre_{s+W-1-j},   dw_j = sum_t dpre_t x_{t-W+1+j},   db = sum_t dpre_t.
//
// HBM-bound: a thread has 16 bytes of neighbouring channels (backward: 4 channels) and walks a run of tokens with the last
// W inputs in registers, so that an input is read once, but for the W - 1 before each run (from L2); the next tokens' loads
// are in flight. The backward forms pre again from x; its dw and db are summed over a run, over the CTA's eight runs in
// shared memory and then over CTAs by a second launch, in a fixed order.
#include "sel_common.cuh"

namespace subq {
namespace {

using sel::Piece;
using sel::need_vec;
using sel::row_of;

constexpr int kConvThreads = 256;
constexpr int kRows = 8;   // backward: runs of a CTA
constexpr int kAhead = 4;  // tokens whose loads are in flight

template <typename T>
__device__ __forceinline__ bool conv_live(const ConvParams& p, int b, int t) {
    return t >= 0 && t < p.L && (!p.mask || p.mask[(int64_t)b * p.mask_sb + t]);
}

// Input of token t (negative: the carried window).
template <typename T, int V, int W>
__device__ __forceinline__ void conv_input(const ConvParams& p, int b, int t, int c, int n, bool vec, bool vec_s, Piece<T, V>& x) {
    if (t < 0) {
        if (p.S_in && t >= 1 - W) x.load(static_cast<const T*>(p.S_in) + ((int64_t)b * (W - 1) + t + W - 1) * p.D + c, n, vec_s);
        else x.zero();
    } else if (conv_live<T>(p, b, t)) {
        x.load(row_of<T>(p.x, b, t, c), n, vec);
    } else {
        x.zero();
    }
}

template <typename T, int V, int W>
struct Taps {
    float w[W][V], bias[V];
    __device__ __forceinline__ void load(const ConvParams& p, int c, int n) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = i < n ? p.w[(int64_t)(c + i) * W + j] : 0.f;
            bias[i] = i < n && p.bias ? p.bias[c + i] : 0.f;
        }
    }
};

template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_fwd_kernel(const ConvParams p, int run, int runs, int keep) {
    const int nv = (p.D + V - 1) / V;
    const int64_t item = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
    if (item >= (int64_t)p.B * runs * nv) return;
    const int c = (int)(item % nv) * V, n = min(V, p.D - c);
    const int64_t r = item / nv;
    const int b = (int)(r / runs), t0 = (int)(r % runs) * run, t1 = min(p.L, t0 + run);
    constexpr int kB = need_vec<V * (int)sizeof(T)>();
    const bool vx = p.x.vec >= kB, vy = p.y.vec >= kB;
    const bool vs = (p.D * (int)sizeof(T)) % kB == 0 && ((reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.S_out)) & (kB - 1)) == 0;
    Taps<T, V, W> tap;
    tap.load(p, c, n);
    float x[W][V];  // the last W inputs, oldest first
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        Piece<T, V> h;
        conv_input<T, V, W>(p, b, t0 - (W - 1) + j, c, n, vx, vs, h);
#pragma unroll
        for (int i = 0; i < V; ++i) x[j + 1][i] = to_f<T>(h.x[i]);
    }
    Piece<T, V> next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) conv_input<T, V, W>(p, b, t0 + k < t1 ? t0 + k : p.L, c, n, vx, vs, next[k]);
    for (int tb = t0; tb < t1; tb += kAhead) {
        Piece<T, V> now[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) now[k] = next[k];
        if (tb + kAhead < t1)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) conv_input<T, V, W>(p, b, tb + kAhead + k < t1 ? tb + kAhead + k : p.L, c, n, vx, vs, next[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int t = tb + k;
            if (t >= t1) break;
            Piece<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) x[j][i] = x[j + 1][i];
                x[W - 1][i] = to_f<T>(now[k].x[i]);
                float s = tap.bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) s = fmaf(tap.w[j][i], x[j][i], s);
                if (p.silu) s *= sel::sigmoid(s);
                o.x[i] = from_f<T>(s);
            }
            if (p.mask && !conv_live<T>(p, b, t)) o.zero();
            o.store(const_cast<T*>(row_of<T>(p.y, b, t, c)), n, vy);
            // the window behind the last token, where no mask ends the sequence before
            if (keep && t >= p.L - (W - 1))
                now[k].store(static_cast<T*>(p.S_out) + ((int64_t)b * (W - 1) + t - (p.L - (W - 1))) * p.D + c, n, vs);
        }
    }
}

// Single tokens and short calls: a thread walks a sequence's channels from the first token to the last.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(const ConvParams p) {
    const int nv = (p.D + V - 1) / V;
    const int64_t item = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
    if (item >= (int64_t)p.B * nv) return;
    const int c = (int)(item % nv) * V, n = min(V, p.D - c), b = (int)(item / nv);
    constexpr int kB = need_vec<V * (int)sizeof(T)>();
    const bool vx = p.x.vec >= kB, vy = p.y.vec >= kB;
    const bool vs = (p.D * (int)sizeof(T)) % kB == 0 && ((reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.S_out)) & (kB - 1)) == 0;
    Taps<T, V, W> tap;
    tap.load(p, c, n);
    Piece<T, V> x[W], kept[W - 1];  // the last W inputs; the window up to the last live token
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        conv_input<T, V, W>(p, b, j - (W - 1), c, n, vx, vs, x[j + 1]);
        kept[j] = x[j + 1];
    }
    for (int t = 0; t < p.L; ++t) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) x[j] = x[j + 1];
        const bool live = conv_live<T>(p, b, t);
        conv_input<T, V, W>(p, b, t, c, n, vx, vs, x[W - 1]);
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = tap.bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) s = fmaf(tap.w[j][i], to_f<T>(x[j].x[i]), s);
            if (p.silu) s *= sel::sigmoid(s);
            o.x[i] = from_f<T>(live ? s : 0.f);
        }
        o.store(const_cast<T*>(row_of<T>(p.y, b, t, c)), n, vy);
        if (live)
#pragma unroll
            for (int j = 0; j < W - 1; ++j) kept[j] = x[j + 1];
    }
    if (p.S_out)
#pragma unroll
        for (int j = 0; j < W - 1; ++j) kept[j].store(static_cast<T*>(p.S_out) + ((int64_t)b * (W - 1) + j) * p.D + c, n, vs);
}

// One past the last live token of a sequence, by all threads of a CTA.
__device__ __forceinline__ int live_end(const uint8_t* mask, int L) {
    int e = 0;
    for (int t = threadIdx.x; t < L; t += kConvThreads)
        if (mask[t]) e = t + 1;
    __shared__ int top;
    if (threadIdx.x == 0) top = 0;
    __syncthreads();
    e = __reduce_max_sync(0xffffffffu, e);
    if ((threadIdx.x & 31) == 0) atomicMax(&top, e);  // (a maximum: any order gives the same)
    __syncthreads();
    return top;
}

// The window behind the last live token (S_out may be S_in: a thread reads its channel's whole window first).
template <typename T, int W>
__global__ void __launch_bounds__(kConvThreads) conv_window_kernel(const ConvParams p) {
    const int b = blockIdx.y, c = blockIdx.x * kConvThreads + threadIdx.x;
    const int e = p.mask ? live_end(p.mask + (int64_t)b * p.mask_sb, p.L) : p.L;
    if (c >= p.D) return;
    Piece<T, 1> x[W - 1];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_input<T, 1, W>(p, b, e - (W - 1) + j, c, 1, false, false, x[j]);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) static_cast<T*>(p.S_out)[((int64_t)b * (W - 1) + j) * p.D + c] = x[j].x[0];
}

__global__ void __launch_bounds__(kConvThreads) conv_ends_kernel(const ConvParams p, int* ends) {
    const int e = live_end(p.mask + (int64_t)blockIdx.x * p.mask_sb, p.L);
    if (threadIdx.x == 0) ends[blockIdx.x] = e;
}

// 32 channel pieces x 8 runs. Gradients of the run's inputs (the first run's: of the carried window, too) and its part of
// dw and db: the tokens behind the run whose taps reach into it are formed again.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_bwd_kernel(const ConvParams p, const int* ends) {
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int c = (blockIdx.x * 32 + lane) * V, n = max(0, min(V, p.D - c));
    const int runs = (p.L + p.run - 1) / p.run;
    const int64_t r = (int64_t)blockIdx.y * kRows + row;
    const bool in = n > 0 && r < (int64_t)p.B * runs;
    constexpr int kB = need_vec<V * (int)sizeof(T)>();
    const bool vx = p.x.vec >= kB, vg = p.dy.vec >= kB, vo = p.dx.vec >= kB;
    const bool vs = (p.D * (int)sizeof(T)) % kB == 0 &&
                    ((reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.dS_out) | reinterpret_cast<uintptr_t>(p.dS_in)) & (kB - 1)) == 0;
    float dw[W][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0.f;
    }
    if (in) {
        const int b = (int)(r / runs), t0 = (int)(r % runs) * p.run, t1 = min(p.L, t0 + p.run);
        const int end = ends ? ends[b] : p.L;
        Taps<T, V, W> tap;
        tap.load(p, c, n);
        float x[W][V], dp[W][V];  // the last W inputs; dpre of the last W tokens
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            Piece<T, V> h;
            conv_input<T, V, W>(p, b, t0 - (W - 1) + j, c, n, vx, vs, h);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[j + 1][i] = to_f<T>(h.x[i]);
                dp[j + 1][i] = 0.f;
            }
        }
        auto load = [&](int t, Piece<T, V>& xs, Piece<T, V>& gs) {
            xs.zero();
            gs.zero();
            if (t < t1 + W - 1 && conv_live<T>(p, b, t)) {
                xs.load(row_of<T>(p.x, b, t, c), n, vx);
                gs.load(row_of<T>(p.dy, b, t, c), n, vg);
            }
        };
        Piece<T, V> nx[kAhead], ng[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load(t0 + k, nx[k], ng[k]);
        for (int tb = t0; tb < t1 + W - 1; tb += kAhead) {
            Piece<T, V> cx[kAhead], cg[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                cx[k] = nx[k];
                cg[k] = ng[k];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) load(tb + kAhead + k, nx[k], ng[k]);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int t = tb + k, s = t - (W - 1);
                if (t >= t1 + W - 1) break;
                Piece<T, V> o;
                float d[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        x[j][i] = x[j + 1][i];
                        dp[j][i] = dp[j + 1][i];
                    }
                    x[W - 1][i] = to_f<T>(cx[k].x[i]);
                    float g = to_f<T>(cg[k].x[i]);  // 0 on tokens that are not live
                    if (p.silu) {
                        float pre = tap.bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) pre = fmaf(tap.w[j][i], x[j][i], pre);
                        const float sg = sel::sigmoid(pre);
                        const float slope = sg * fmaf(pre, 1.f - sg, 1.f);
                        g = conv_live<T>(p, b, t) ? g * slope : 0.f;
                    }
                    dp[W - 1][i] = g;
                    if (t < t1) {
                        db[i] += g;
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[j][i] = fmaf(g, x[j][i], dw[j][i]);
                    }
                    d[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < W; ++j) d[i] = fmaf(tap.w[j][i], dp[W - 1 - j][i], d[i]);
                }
                // (the run before this one, whose last tokens these are, writes tokens before t0)
                if (s < t0 && !(t0 == 0 && p.dS_in)) continue;
                const int at = s - end + W - 1;  // its place in the window that was handed on
                if (p.dS_out && at >= 0 && at < W - 1) {
                    Piece<T, V> h;
                    h.load(static_cast<const T*>(p.dS_out) + ((int64_t)b * (W - 1) + at) * p.D + c, n, vs);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] += to_f<T>(h.x[i]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) o.x[i] = from_f<T>(s < 0 || conv_live<T>(p, b, s) ? d[i] : 0.f);
                if (s >= 0) o.store(const_cast<T*>(row_of<T>(p.dx, b, s, c)), n, vo);
                else o.store(static_cast<T*>(p.dS_in) + ((int64_t)b * (W - 1) + s + W - 1) * p.D + c, n, vs);
            }
        }
    }
    __shared__ float red[kRows][W + 1][32 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        red[row][W][lane * V + i] = db[i];
#pragma unroll
        for (int j = 0; j < W; ++j) red[row][j][lane * V + i] = dw[j][i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (W + 1) * 32 * V; i += kConvThreads) {
        const int j = i / (32 * V), at = i % (32 * V), ch = blockIdx.x * 32 * V + at;
        if (ch >= p.D) continue;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) s += red[k][j][at];
        p.part[((int64_t)blockIdx.y * (W + 1) + j) * p.D + ch] = s;
    }
}

__device__ __forceinline__ void add_kept(float& s, float& rest, float x) {
    const float t = __fadd_rn(s, x), z = __fsub_rn(t, s);
    rest = __fadd_rn(rest, __fadd_rn(__fsub_rn(s, __fsub_rn(t, z)), __fsub_rn(x, z)));
    s = t;
}

__global__ void __launch_bounds__(kConvThreads) conv_sum_kernel(const ConvParams p) {
    const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31), n = (int64_t)(p.W + 1) * p.D;
    const int part = threadIdx.x >> 5;  // eight threads for one value, each with every eighth part
    float s = 0.f, rest = 0.f;
    if (i < n)
#pragma unroll 4
        for (int k = part; k < p.parts; k += 8) add_kept(s, rest, p.part[k * n + i]);
    __shared__ float red[8][32];
    red[part][threadIdx.x & 31] = s + rest;
    __syncthreads();
    if (part || i >= n) return;
    s = rest = 0.f;
    for (int k = 0; k < 8; ++k) add_kept(s, rest, red[k][threadIdx.x]);
    const int j = (int)(i / p.D), c = (int)(i % p.D);
    if (j < p.W) p.dw[(int64_t)c * p.W + j] = s + rest;
    else if (p.db) p.db[c] = s + rest;
}

// The widest pieces that the rows' alignment allows, or single channels.
template <typename T>
bool pieces_fit(const ConvParams& p, bool bwd) {
    const int need = bwd ? 4 * (int)sizeof(T) : 16;
    return bwd ? p.x.vec >= need && p.dy.vec >= need && p.dx.vec >= need : p.x.vec >= need && p.y.vec >= need;
}

template <typename T, int V, int W>
cudaError_t conv_fwd(const ConvParams& p, cudaStream_t st, int* launches) {
    const int64_t nv = (p.D + V - 1) / V;
    auto blocks = [](int64_t n) { return (unsigned)((n + kConvThreads - 1) / kConvThreads); };
    if (p.L <= 8) {
        conv_step_kernel<T, V, W><<<blocks(p.B * nv), kConvThreads, 0, st>>>(p);
        *launches = 1;
        return cudaGetLastError();
    }
    const int run = (int64_t)p.B * p.L * nv >= (int64_t)148 * 2048 * 16 ? 32 : 16;
    const int runs = (p.L + run - 1) / run, keep = p.S_out && !p.mask && p.S_out != p.S_in && p.L >= W - 1;
    conv_fwd_kernel<T, V, W><<<blocks((int64_t)p.B * runs * nv), kConvThreads, 0, st>>>(p, run, runs, keep);
    *launches = 1;
    if (p.S_out && !keep) {
        conv_window_kernel<T, W><<<dim3(blocks(p.D), p.B), kConvThreads, 0, st>>>(p);
        *launches = 2;
    }
    return cudaGetLastError();
}

template <typename T, int V, int W>
cudaError_t conv_bwd(const ConvParams& p, cudaStream_t st, int* launches) {
    *launches = 2;
    const int* ends = nullptr;
    if (p.dS_out && p.mask) {
        int* at = reinterpret_cast<int*>(p.part + (int64_t)p.parts * (W + 1) * p.D);
        conv_ends_kernel<<<p.B, kConvThreads, 0, st>>>(p, at);
        ends = at;
        *launches = 3;
    }
    conv_bwd_kernel<T, V, W><<<dim3((p.D + 32 * V - 1) / (32 * V), p.parts), kConvThreads, 0, st>>>(p, ends);
    conv_sum_kernel<<<(unsigned)(((int64_t)(W + 1) * p.D + 31) / 32), kConvThreads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t conv_any(const ConvParams& p, bool bwd, cudaStream_t st, int* launches) {
    auto width = [&](auto v) {
        constexpr int V = decltype(v)::value, B = V == 1 ? 1 : 4;
        switch (p.W) {
            case 2: return bwd ? conv_bwd<T, B, 2>(p, st, launches) : conv_fwd<T, V, 2>(p, st, launches);
            case 3: return bwd ? conv_bwd<T, B, 3>(p, st, launches) : conv_fwd<T, V, 3>(p, st, launches);
            default: return bwd ? conv_bwd<T, B, 4>(p, st, launches) : conv_fwd<T, V, 4>(p, st, launches);
        }
    };
    return pieces_fit<T>(p, bwd) ? width(std::integral_constant<int, 16 / (int)sizeof(T)>{}) : width(std::integral_constant<int, 1>{});
}

cudaError_t conv_typed(const ConvParams& p, int dtype, bool bwd, cudaStream_t st, int* launches) {
    return dtype == SUBQ_BF16 ? conv_any<__nv_bfloat16>(p, bwd, st, launches)
                              : dtype == SUBQ_FP16 ? conv_any<__half>(p, bwd, st, launches) : conv_any<float>(p, bwd, st, launches);
}

}  // namespace

cudaError_t launch_conv_fwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches) { return conv_typed(p, dtype, false, st, launches); }
cudaError_t launch_conv_bwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches) { return conv_typed(p, dtype, true, st, launches); }

void conv_bwd_split(ConvParams& p) {
    p.run = 32;
    for (;; p.run *= 2) {  // (a grid has at most 65535 rows of CTAs)
        const int64_t runs = (int64_t)p.B * ((p.L + p.run - 1) / p.run), parts = (runs + kRows - 1) / kRows;
        p.parts = (int)parts;
        if (parts <= 65535) return;
    }
}

}  // namespace subq
