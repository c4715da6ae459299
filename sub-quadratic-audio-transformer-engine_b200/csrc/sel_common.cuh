// Shared device code of the selective scan. Per channel d and state n
//   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = sum_n C_t h_t + D u_t,   out_t = y_t silu(z_t),
// dt_t = softplus(raw_t + bias). A channel's states lie four to a lane on LPC lanes (4, 8, 16 or 32: up to 16, 32, 64, 128
// states), so that B and C are read as 16-byte pieces that every channel of a warp shares, and y is a sum over LPC lanes.
//
// A step multiplies by a = exp(dt A). Rounded by itself an a near 1 is off by up to 2^-25 the same way at every token, and
// the state remembers 1 / (1 - a) of them; so the step is h + (a - 1) h, with a - 1 = 2^y - 1 (y = dt A log2 e) from a
// polynomial where |y| < 1/4 (Chebyshev fit of (2^y - 1) / y, 2e-8 off), and from the exponential unit beyond, where the
// state remembers six tokens.
#pragma once

#include <type_traits>

#include "block_launch.h"
#include "scan_common.cuh"

namespace subq {
namespace sel {

// Two float32 in a 64-bit register: one instruction for two multiplications.
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ void get(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ float both(F2 x) {
    float a, b;
    get(x, a, b);
    return a + b;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

constexpr float kNear = 0.25f;
// 2^y - 1.
__device__ __forceinline__ F2 decay(F2 y) {
    F2 p = fma(y, f2(0.0013347864f), f2(0.00963017f));
    p = fma(p, y, f2(0.055504076f));
    p = fma(p, y, f2(0.24022631f));
    p = fma(p, y, f2(0.6931472f));
    p = mul(p, y);
    float y0, y1, p0, p1, e0, e1;
    get(y, y0, y1);
    get(p, p0, p1);
    get(add(f2(ex2(y0), ex2(y1)), f2(-1.f)), e0, e1);
    return f2(fabsf(y0) < kNear ? p0 : e0, fabsf(y1) < kNear ? p1 : e1);
}
__device__ __forceinline__ float decay(float y) {
    float p = fmaf(y, 0.0013347864f, 0.00963017f);
    p = fmaf(p, y, 0.055504076f);
    p = fmaf(p, y, 0.24022631f);
    p = fmaf(p, y, 0.6931472f) * y;
    return fabsf(y) < kNear ? p : ex2(y) - 1.f;
}

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }
__device__ __forceinline__ float sigmoid(float x) {  // from exp(-|x|), so that neither side overflows
    const float e = expf(-fabsf(x)), r = __fdividef(1.f, 1.f + e);
    return x >= 0.f ? r : e * r;
}

// Sums v[0..3] over the LPC lanes of a channel: lane q of them (q < 4) has the sum of v[q].
template <int LPC>
__device__ __forceinline__ float lane_sums4(const float (&v)[4], int lane) {
    const bool b0 = lane & 1, b1 = lane & 2;
    float a = b0 ? v[1] : v[0], c = b0 ? v[3] : v[2];
    a += __shfl_xor_sync(0xffffffffu, b0 ? v[0] : v[1], 1);
    c += __shfl_xor_sync(0xffffffffu, b0 ? v[2] : v[3], 1);
    float s = b1 ? c : a;
    s += __shfl_xor_sync(0xffffffffu, b1 ? a : c, 2);
#pragma unroll
    for (int o = 4; o < LPC; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// V consecutive elements of a row in one access where `vec` bytes allow it.
template <typename T, int V>
struct Piece {
    T x[V];
    __device__ __forceinline__ void load(const T* at, int n, bool vec) {
        constexpr int kB = V * (int)sizeof(T);
        if (vec && n >= V) {
            if constexpr (kB >= 16) {
#pragma unroll
                for (int i = 0; i < kB / 16; ++i) reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(at)[i];
            } else if constexpr (kB == 8) {
                *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(at);
            } else if constexpr (kB == 4) {
                *reinterpret_cast<uint32_t*>(x) = *reinterpret_cast<const uint32_t*>(at);
            } else {
                x[0] = at[0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = i < n ? at[i] : from_f<T>(0.f);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = from_f<T>(0.f);
    }
    __device__ __forceinline__ void store(T* at, int n, bool vec) const {
        constexpr int kB = V * (int)sizeof(T);
        if (vec && n >= V) {
            if constexpr (kB >= 16) {
#pragma unroll
                for (int i = 0; i < kB / 16; ++i) reinterpret_cast<uint4*>(at)[i] = reinterpret_cast<const uint4*>(x)[i];
            } else if constexpr (kB == 8) {
                *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(x);
            } else if constexpr (kB == 4) {
                *reinterpret_cast<uint32_t*>(at) = *reinterpret_cast<const uint32_t*>(x);
            } else {
                at[0] = x[0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) at[i] = x[i];
        }
    }
};
template <int B>
__host__ __device__ constexpr int need_vec() {
    return B > 16 ? 16 : B;
}

// Which channels and tokens a CTA has, and what of it a thread stages: row `row` of a tile, V channels from `c0`.
template <typename T, int LPC>
struct Place {
    static constexpr int kCh = kSelThreads / LPC, kV = kSelTile * kCh / kSelThreads, kPer = kCh / kV;  // channels; staged at once; threads a row
    int b, g, d0, nch;  // sequence, group, first channel, live channels of this CTA
    int row, c0, left;  // staging: row, first channel, live channels from there
    __device__ __forceinline__ Place(const SelParams& p) {
        const int blocks = (p.Dg + kCh - 1) / kCh;
        const int x = blockIdx.x;
        b = x / (blocks * p.G);
        g = x / blocks % p.G;
        const int k = x % blocks;
        d0 = g * p.Dg + k * kCh;
        nch = min(kCh, p.Dg - k * kCh);
        row = threadIdx.x / kPer;
        c0 = threadIdx.x % kPer * kV;
        left = max(0, min(kV, nch - c0));
    }
    __device__ __forceinline__ int block(const SelParams& p) const { return blockIdx.x % ((p.Dg + kCh - 1) / kCh); }
};
template <typename T>
__device__ __forceinline__ const T* row_of(const SelTensor& t, int b, int l, int d) {
    return static_cast<const T*>(t.p) + b * t.sb + l * t.sl + d;
}
template <typename T>
__device__ __forceinline__ bool live_at(const SelParams& p, int b, int l) {
    return l < p.L && (!p.mask || p.mask[(int64_t)b * p.mask_sb + l]);
}

// A tile's rows of B or C as float32, zeros on masked tokens, behind the last token and behind the N-th state.
template <typename T, int LPC>
struct States {
    static constexpr int kNp = 4 * LPC, kPer = kSelTile * kNp / kSelThreads;
    T x[kPer];
    __device__ __forceinline__ void load(const SelParams& p, const SelTensor& t, int b, int g, int l0, int l1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = threadIdx.x + i * kSelThreads, l = l0 + at / kNp, n = at % kNp;
            const bool in = n < p.N && l < l1 && live_at<T>(p, b, l);
            x[i] = in ? (static_cast<const T*>(t.p) + b * t.sb + l * t.sl + g * t.sg)[n] : from_f<T>(0.f);
        }
    }
    __device__ __forceinline__ void put(float* to) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) to[threadIdx.x + i * kSelThreads] = to_f<T>(x[i]);
    }
};

}  // namespace sel
}  // namespace subq
