// Short causal convolution over [B, L, D], one filter of W = 2, 3 or 4 taps a channel, forward and backward:
//   pre_t = b + sum_j w_j x_{t-W+1+j},   y_t = silu(pre_t) or pre_t.
// Before the first token stands the carried window (the W - 1 inputs before it, zeros without one); a masked token's input
// counts as 0 and its output is 0; the window that is handed on is of the W - 1 inputs up to the last live token.
//   dpre_t = dy_t act'(pre_t),   dx_s = sum_j w_j dpre_{s+W-1-j},   dw_j = sum_t dpre_t x_{t-W+1+j},   db = sum_t dpre_t.
//
// HBM-bound: a thread has four neighbouring channels (backward: two; single ones where rows are not aligned) and a
// run of eight tokens (backward: sixteen), all of whose rows it asks for at once, those of the tokens that its taps reach into among them (L1 has
// them for the CTA's next run). The backward forms pre again from x; its dw and db are summed over a run, over the CTA's
// eight runs in shared memory and then over CTAs by a second launch, in a fixed order.
// 8 x 2047 x 1536 in bf16: forward 35 us (HBM floor 15; its warps wait for their rows: a thread loads its run, computes and ends),
// backward 86 us (23; float32 94: nineteen sums before the activation for sixteen tokens, and its derivative, at 15 warps an SM
// that wait for the instruction before). Issue slots are 0.6 used in both.
#include <algorithm>

#include "sel_common.cuh"

namespace subq {
namespace {

using sel::Piece;
using sel::row_of;

constexpr int kConvThreads = 256;
constexpr int kRun = 8;   // tokens of a thread
constexpr int kBack = 16;  // the same, backward (eight, at three CTAs an SM: 150 us for 133 of a step of 8 x 2047 x 1536)
constexpr int kRows = 8;  // runs of a CTA, one after another

template <typename T>
__device__ __forceinline__ bool conv_live(const ConvParams& p, int b, int t) {
    return t >= 0 && t < p.L && (!p.mask || p.mask[(int64_t)b * p.mask_sb + t]);
}

// Input of token t (negative: the carried window). What a masked token holds is loaded, but not used.
template <typename T, int V, int W>
__device__ __forceinline__ void conv_input(const ConvParams& p, int b, int t, int c, Piece<T, V>& x) {
    x.zero();
    if (t < 0) {
        if (p.S_in && t >= 1 - W) x.load(static_cast<const T*>(p.S_in) + ((int64_t)b * (W - 1) + t + W - 1) * p.D + c);
    } else if (t < p.L) {
        const bool live = conv_live<T>(p, b, t);
        x.load(row_of<T>(p.x, b, t, c));
        if (!live) x.zero();
    }
}

using sel::F2;
using sel::f2;

// A thread's channels two at a time (a single one beside a 0).
template <typename T, int V>
__device__ __forceinline__ void to_pairs(const Piece<T, V>& x, F2 (&f)[(V + 1) / 2]) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) f[i] = f2(to_f<T>(x.x[2 * i]), V > 1 ? to_f<T>(x.x[2 * i + (V > 1)]) : 0.f);
}
template <typename T, int V>
__device__ __forceinline__ void from_pairs(const F2 (&f)[(V + 1) / 2], Piece<T, V>& x) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) {
        float a, b;
        sel::get(f[i], a, b);
        x.x[2 * i] = from_f<T>(a);
        if (V > 1) x.x[2 * i + (V > 1)] = from_f<T>(b);
    }
}

template <typename T, int V, int W>
struct Taps {
    static constexpr int H = (V + 1) / 2;
    F2 w[W][H], bias[H];
    __device__ __forceinline__ void load(const ConvParams& p, int c) {
        constexpr int kAll = V * W;
        float x[2 * H * W];
        if (kAll % 4 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0) {  // (c is a multiple of V)
#pragma unroll
            for (int i = 0; i < kAll / 4; ++i) {
                const float4 v = reinterpret_cast<const float4*>(p.w + (int64_t)c * W)[i];
                x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kAll; ++i) x[i] = p.w[(int64_t)c * W + i];
        }
        if (V == 1)
#pragma unroll
            for (int j = 0; j < W; ++j) x[W + j] = 0.f;
#pragma unroll
        for (int i = 0; i < H; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = f2(x[2 * i * W + j], x[(2 * i + 1) * W + j]);
            bias[i] = p.bias ? f2(p.bias[c + 2 * i], V > 1 ? p.bias[c + 2 * i + (V > 1)] : 0.f) : f2(0.f);
        }
    }
};

// Rows t0 .. t0 + M - 1 of a tensor, all asked for before the first is used (a run at an end of the sequence asks one by one).
template <typename T, int V, int M>
__device__ __forceinline__ void load_rows(const SelTensor& x, int L, int b, int t0, int c, Piece<T, V>* to) {
    if (t0 >= 0 && t0 + M <= L) {
        const T* at = row_of<T>(x, b, t0, c);
#pragma unroll
        for (int k = 0; k < M; ++k) to[k].load(at + k * x.sl);
    } else {
#pragma unroll
        for (int k = 0; k < M; ++k) {
            to[k].zero();
            if (t0 + k >= 0 && t0 + k < L) to[k].load(row_of<T>(x, b, t0 + k, c));
        }
    }
}
// Which of them are live, a bit each; rows before the first token are.
template <int M>
__device__ __forceinline__ uint32_t live_rows(const ConvParams& p, int b, int t0) {
    uint32_t live = 0;
    if (!p.mask) {
#pragma unroll
        for (int k = 0; k < M; ++k) live |= t0 + k < p.L ? 1u << k : 0u;
        return live;
    }
    const uint8_t* at = p.mask + (int64_t)b * p.mask_sb;
    uint8_t m[M];
#pragma unroll
    for (int k = 0; k < M; ++k) m[k] = at[min(max(t0 + k, 0), p.L - 1)];
#pragma unroll
    for (int k = 0; k < M; ++k) live |= t0 + k < 0 || (m[k] && t0 + k < p.L) ? 1u << k : 0u;
    return live;
}
template <typename T, int V, int W>
__device__ __forceinline__ void load_window(const ConvParams& p, int b, int t0, int c, Piece<T, V>* to) {
    if (t0 != 0 || !p.S_in) return;  // (runs are longer than a window)
#pragma unroll
    for (int k = 0; k < W - 1; ++k) to[k].load(static_cast<const T*>(p.S_in) + ((int64_t)b * (W - 1) + k) * p.D + c);
}

// 32 channel pieces x 8 runs a CTA.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads, 4) conv_fwd_kernel(const ConvParams p, int runs, int across, int keep) {
    const int group = blockIdx.x / across, c = ((blockIdx.x - group * across) * 32 + (threadIdx.x & 31)) * V;
    const int64_t r = (int64_t)group * kRows + (threadIdx.x >> 5);
    if (c >= p.D || r >= (int64_t)p.B * runs) return;
    const int b = (int)(r / runs), t0 = (int)(r - (int64_t)b * runs) * kRun;
    Piece<T, V> x[W - 1 + kRun];
    load_rows<T, V, W - 1 + kRun>(p.x, p.L, b, t0 - (W - 1), c, x);
    load_window<T, V, W>(p, b, t0, c, x);
    const uint32_t live = live_rows<W - 1 + kRun>(p, b, t0 - (W - 1));
    Taps<T, V, W> tap;
    tap.load(p, c);
    constexpr int H = (V + 1) / 2;
    F2 f[W - 1 + kRun][H];
    // (a row is a warp's: whether its token is live is no divergence)
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        if (!(live >> k & 1)) x[k].zero();
        to_pairs(x[k], f[k]);
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        const int t = t0 + k;
        if (t >= p.L) break;
        Piece<T, V>& now = x[k + W - 1];
        const bool on = live >> (k + W - 1) & 1;
        if (!on) now.zero();
        to_pairs(now, f[k + W - 1]);
        Piece<T, V> o;
        o.zero();
        if (on) {
            F2 s[H];
#pragma unroll
            for (int i = 0; i < H; ++i) {
                s[i] = tap.bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) s[i] = sel::fma(tap.w[j][i], f[k + j][i], s[i]);
                if (p.silu) s[i] = sel::mul(s[i], sel::sigmoid(s[i]));
            }
            from_pairs(s, o);
        }
        o.store(const_cast<T*>(row_of<T>(p.y, b, t, c)));
        // the window behind the last token, where no mask ends the sequence before
        if (keep && t >= p.L - (W - 1)) now.store(static_cast<T*>(p.S_out) + ((int64_t)b * (W - 1) + t - (p.L - (W - 1))) * p.D + c);
    }
}

// Single tokens and short calls: a thread walks a sequence's channels from the first token to the last.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(const ConvParams p) {
    const int nv = (p.D + V - 1) / V;
    const int64_t item = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
    if (item >= (int64_t)p.B * nv) return;
    const int c = (int)(item % nv) * V, b = (int)(item / nv);
    Taps<T, V, W> tap;
    tap.load(p, c);
    Piece<T, V> x[W], kept[W - 1];  // the last W inputs; the window up to the last live token
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        conv_input<T, V, W>(p, b, j - (W - 1), c, x[j + 1]);
        kept[j] = x[j + 1];
    }
    for (int t = 0; t < p.L; ++t) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) x[j] = x[j + 1];
        const bool live = conv_live<T>(p, b, t);
        conv_input<T, V, W>(p, b, t, c, x[W - 1]);
        Piece<T, V> o;
        constexpr int H = (V + 1) / 2;
        F2 s[H];
#pragma unroll
        for (int i = 0; i < H; ++i) s[i] = tap.bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            F2 f[H];
            to_pairs(x[j], f);
#pragma unroll
            for (int i = 0; i < H; ++i) s[i] = sel::fma(tap.w[j][i], f[i], s[i]);
        }
        if (p.silu)
#pragma unroll
            for (int i = 0; i < H; ++i) s[i] = sel::mul(s[i], sel::sigmoid(s[i]));
        from_pairs(s, o);
        if (!live) o.zero();
        o.store(const_cast<T*>(row_of<T>(p.y, b, t, c)));
        if (live)
#pragma unroll
            for (int j = 0; j < W - 1; ++j) kept[j] = x[j + 1];
    }
    if (p.S_out)
#pragma unroll
        for (int j = 0; j < W - 1; ++j) kept[j].store(static_cast<T*>(p.S_out) + ((int64_t)b * (W - 1) + j) * p.D + c);
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
    for (int j = 0; j < W - 1; ++j) conv_input<T, 1, W>(p, b, e - (W - 1) + j, c, x[j]);
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
__global__ void __launch_bounds__(kConvThreads, 2) conv_bwd_kernel(const ConvParams p, const int* ends) {
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int c = (blockIdx.x * 32 + lane) * V;
    const int runs = (p.L + kBack - 1) / kBack;
    constexpr int kTail = kBack + W - 1;
    constexpr int H = (V + 1) / 2;
    F2 dw[W][H], db[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
        db[i] = f2(0.f);
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = f2(0.f);
    }
    for (int turn = 0; turn < p.run; ++turn) {  // groups of eight runs
        const int64_t r = ((int64_t)blockIdx.y * p.run + turn) * kRows + row;
        if (c >= p.D || r >= (int64_t)p.B * runs) break;
        const int b = (int)(r / runs), t0 = (int)(r - (int64_t)b * runs) * kBack, t1 = min(p.L, t0 + kBack);
        const int end = p.dS_out ? ends ? ends[b] : p.L : 0;
        // tokens t0 - (W - 1) .. t0 + kBack + W - 2 of x, t0 .. of dy: the taps of the last ones reach into the run
        Piece<T, V> x[W - 1 + kTail], g[kTail];
        load_rows<T, V, W - 1 + kTail>(p.x, p.L, b, t0 - (W - 1), c, x);
        load_rows<T, V, kTail>(p.dy, p.L, b, t0, c, g);
        load_window<T, V, W>(p, b, t0, c, x);
        const uint32_t live = live_rows<W - 1 + kTail>(p, b, t0 - (W - 1));
        Taps<T, V, W> tap;
        tap.load(p, c);
        F2 f[W - 1 + kTail][H], dp[W - 1 + kTail][H];  // inputs; dpre, 0 before the run
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            if (!(live >> k & 1)) x[k].zero();
            to_pairs(x[k], f[k]);
#pragma unroll
            for (int i = 0; i < H; ++i) dp[k][i] = f2(0.f);
        }
#pragma unroll
        for (int k = 0; k < kTail; ++k) {
            const int at = k + W - 1;
            const bool on = live >> at & 1;
            if (!on) x[at].zero();
            to_pairs(x[at], f[at]);
#pragma unroll
            for (int i = 0; i < H; ++i) dp[at][i] = f2(0.f);
            if (on) {
                to_pairs(g[k], dp[at]);
                if (p.silu)
#pragma unroll
                    for (int i = 0; i < H; ++i) {
                        F2 pre = tap.bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) pre = sel::fma(tap.w[j][i], f[k + j][i], pre);
                        const F2 sg = sel::sigmoid(pre);  // silu' = sg (1 + pre (1 - sg))
                        dp[at][i] = sel::mul(dp[at][i], sel::mul(sg, sel::fma(pre, sel::fma(sg, f2(-1.f), f2(1.f)), f2(1.f))));
                    }
                if (k < kBack)
#pragma unroll
                    for (int i = 0; i < H; ++i) {
                        db[i] = sel::add(db[i], dp[at][i]);
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[j][i] = sel::fma(dp[at][i], f[k + j][i], dw[j][i]);
                    }
            }
            // token s, whose taps have all been seen (before the run's first: the carried window's, of the first run)
            const int s = t0 + k - (W - 1);
            if (s >= t1 || (k < W - 1 && !(t0 == 0 && p.dS_in))) continue;
            F2 d[H];
#pragma unroll
            for (int i = 0; i < H; ++i) {
                d[i] = f2(0.f);
#pragma unroll
                for (int j = 0; j < W; ++j) d[i] = sel::fma(tap.w[j][i], dp[at - j][i], d[i]);
            }
            const int place = s - end + W - 1;  // in the window that was handed on
            if (p.dS_out && place >= 0 && place < W - 1) {
                Piece<T, V> h;
                F2 more[H];
                h.load(static_cast<const T*>(p.dS_out) + ((int64_t)b * (W - 1) + place) * p.D + c);
                to_pairs(h, more);
#pragma unroll
                for (int i = 0; i < H; ++i) d[i] = sel::add(d[i], more[i]);
            }
            Piece<T, V> o;
            from_pairs(d, o);
            if (!(live >> k & 1)) o.zero();
            if (k >= W - 1) o.store(const_cast<T*>(row_of<T>(p.dx, b, s, c)));
            else o.store(static_cast<T*>(p.dS_in) + ((int64_t)b * (W - 1) + s + W - 1) * p.D + c);
        }
    }
    __shared__ float red[kRows][W + 1][32 * V];
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
        for (int j = 0; j <= W; ++j) {
            float a, b;
            sel::get(j < W ? dw[j < W ? j : 0][i] : db[i], a, b);
            red[row][j][lane * V + 2 * i] = a;
            if (V > 1) red[row][j][lane * V + 2 * i + (V > 1)] = b;
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

// Channels of a thread: four, or two in the backward, whose sixteen tokens of four channels do not fit the registers (float32
// training step, us, of four and two: 8 x 2047 x 1536, W = 4, padded 179, 150; 16 x 2048 x 1024, W = 3 205, 150, W = 2 174, 146;
// 4 x 2000 x 1022 88 (single ones), 67; 4 x 1024 x 768 44, 44).
constexpr int pieces(bool bwd) { return bwd ? 2 : 4; }
// Do the channels come out even, and all rows' alignments allow them?
template <typename T>
bool pieces_fit(const ConvParams& p, bool bwd) {
    const int n = pieces(bwd), need = n * (int)sizeof(T);
    const uintptr_t windows = bwd ? reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.dS_out) | reinterpret_cast<uintptr_t>(p.dS_in)
                                  : reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.S_out);
    if (p.D % n || windows % need || p.x.vec < need) return false;
    return bwd ? p.dy.vec >= need && p.dx.vec >= need : p.y.vec >= need;
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
    const int runs = (p.L + kRun - 1) / kRun, keep = p.S_out && !p.mask && p.S_out != p.S_in && p.L >= W - 1;
    const int across = (int)((nv + 31) / 32);
    conv_fwd_kernel<T, V, W><<<(unsigned)(((int64_t)p.B * runs + kRows - 1) / kRows * across), kConvThreads, 0, st>>>(p, runs, across, keep);
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
    auto width = [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (bwd) return pieces_fit<T>(p, true) ? conv_bwd<T, pieces(true), W>(p, st, launches) : conv_bwd<T, 1, W>(p, st, launches);
        return pieces_fit<T>(p, false) ? conv_fwd<T, pieces(false), W>(p, st, launches) : conv_fwd<T, 1, W>(p, st, launches);
    };
    if (p.W == 2) return width(std::integral_constant<int, 2>{});
    return p.W == 3 ? width(std::integral_constant<int, 3>{}) : width(std::integral_constant<int, 4>{});
}

cudaError_t conv_typed(const ConvParams& p, int dtype, bool bwd, cudaStream_t st, int* launches) {
    return dtype == SUBQ_BF16 ? conv_any<__nv_bfloat16>(p, bwd, st, launches)
                              : dtype == SUBQ_FP16 ? conv_any<__half>(p, bwd, st, launches) : conv_any<float>(p, bwd, st, launches);
}

}  // namespace

cudaError_t launch_conv_fwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches) { return conv_typed(p, dtype, false, st, launches); }
cudaError_t launch_conv_bwd(const ConvParams& p, int dtype, cudaStream_t st, int* launches) { return conv_typed(p, dtype, true, st, launches); }

// Groups of eight runs that a CTA goes through: one for each place on the card (two CTAs an SM) or so, so that there are few
// partial sums (and a grid has at most 65535 rows of CTAs).
void conv_bwd_split(ConvParams& p) {
    const int64_t groups = ((int64_t)p.B * ((p.L + kBack - 1) / kBack) + kRows - 1) / kRows, across = (p.D + 63) / 64;
    const int64_t places = std::max<int64_t>(1, 4 * 296 / across);
    p.run = (int)std::max<int64_t>(1, std::max((groups + 65534) / 65535, groups / places));
    p.parts = (int)((groups + p.run - 1) / p.run);
}

}  // namespace subq
