// Shared device code of the selective scan. Per channel d and state n
//   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = sum_n C_t h_t + D u_t,   out_t = y_t silu(z_t),
// dt_t = softplus(raw_t + bias). A channel's states lie four to a lane on LPC lanes (4, 8, 16 or 32: up to 16, 32, 64, 128
// states), so that B and C are read as 16-byte pieces that every channel of a warp shares, and y is a sum over LPC lanes.
//
// A step multiplies by a = exp(dt A) = 2^y. Rounded by itself an a near 1 is off by up to 2^-25 the same way at every token,
// and the state remembers 1 / (1 - a) of them; so where |y| < 1/4 the step is h + (a - 1) h with a - 1 from a polynomial
// (Chebyshev fit of (2^y - 1) / y, 2e-8 off). Beyond, where the state remembers six tokens, it is a h with a from the
// exponential unit (1e-7 off), which a - 1 would leave no bits of a small a.
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
// A step's factor: 2^y - 1 where y is near 0, 2^y beyond.
struct Factor {
    F2 c;
    bool n0, n1;
};
__device__ __forceinline__ Factor factor(F2 y) {
    F2 p = fma(y, f2(0.0013347864f), f2(0.00963017f));
    p = fma(p, y, f2(0.055504076f));
    p = fma(p, y, f2(0.24022631f));
    p = fma(p, y, f2(0.6931472f));
    p = mul(p, y);
    float y0, y1, p0, p1;
    get(y, y0, y1);
    get(p, p0, p1);
    Factor r;
    r.n0 = fabsf(y0) < kNear;
    r.n1 = fabsf(y1) < kNear;
    const float e0 = ex2(y0), e1 = ex2(y1);
    r.c = f2(r.n0 ? p0 : e0, r.n1 ? p1 : e1);
    return r;
}
// a h.
__device__ __forceinline__ F2 decayed(const Factor& f, F2 h) {
    float h0, h1;
    get(h, h0, h1);
    return fma(f.c, h, f2(f.n0 ? h0 : 0.f, f.n1 ? h1 : 0.f));
}
// Factors over many tokens where states grow (A above 0): 2^y beyond 2^127 goes in two steps, so that what is 0 stays 0.
__device__ __forceinline__ float split_growth(float& y, float h) {
    if (y > 127.f) {
        h *= ex2(fminf(y, 254.f) - 127.f);
        y = 127.f;
    }
    return h;
}
__device__ __forceinline__ float decayed(float y, float h) {
    float p = fmaf(y, 0.0013347864f, 0.00963017f);
    p = fmaf(p, y, 0.055504076f);
    p = fmaf(p, y, 0.24022631f);
    p = fmaf(p, y, 0.6931472f) * y;
    p = fmaf(p, h, h);
    const bool near = fabsf(y) < kNear;
    h = split_growth(y, h);
    return near ? p : ex2(y) * h;
}

__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// -|x|, -128 beyond it, where exp is 0 in float32 (products of an infinite or the lowest x would be inf - inf); a NaN stays one.
__device__ __forceinline__ float far_neg(float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(-fabsf(x)), "f"(-128.f));
    return r;
}
// exp(-|x|): the product with log2 e is carried to 48 bits, so that a far x costs no accuracy (3e-7 off at most).
__device__ __forceinline__ float exp_neg(float x) {
    const float a = far_neg(x), t = a * 1.4426950408889634f;
    const float rest = fmaf(a, 1.4426950408889634f, -t);
    const float e = ex2(t);
    return fmaf(e * 0.6931472f, fmaf(a, 1.925963033e-8f, rest), e);
}
// max(x, 0) + log(1 + exp(-|x|)); log(1 + e) / e by a Chebyshev fit of degree 8 on [0, 1] (3e-8 off), accurate for small e.
__device__ __forceinline__ float softplus(float x) {
    const float e = exp_neg(x);
    float p = fmaf(e, 0.005253458f, -0.029588507f);
    p = fmaf(p, e, 0.07836167f);
    p = fmaf(p, e, -0.1367477f);
    p = fmaf(p, e, 0.1911143f);
    p = fmaf(p, e, -0.2484437f);
    p = fmaf(p, e, 0.3331927f);
    p = fmaf(p, e, -0.49999502f);
    p = fmaf(p, e, 1.f);
    return fmaf(p, e, fmaxf(x, 0.f));
}
// 1 / (1 + exp(-x)); an overflow of exp(-x) gives 0.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(x * -1.4426950408889634f)); }

// The same for two.
__device__ __forceinline__ F2 exp_neg(F2 x) {
    float a, b;
    get(x, a, b);
    const F2 m = f2(far_neg(a), far_neg(b)), t = mul(m, f2(1.4426950408889634f));
    F2 rest = fma(m, f2(1.4426950408889634f), mul(t, f2(-1.f)));
    rest = fma(m, f2(1.925963033e-8f), rest);
    get(t, a, b);
    const F2 e = f2(ex2(a), ex2(b));
    return fma(mul(e, f2(0.6931472f)), rest, e);
}
// (e: exp(-|x|))
__device__ __forceinline__ F2 softplus(F2 x, F2& e) {
    e = exp_neg(x);
    F2 p = fma(e, f2(0.005253458f), f2(-0.029588507f));
    p = fma(p, e, f2(0.07836167f));
    p = fma(p, e, f2(-0.1367477f));
    p = fma(p, e, f2(0.1911143f));
    p = fma(p, e, f2(-0.2484437f));
    p = fma(p, e, f2(0.3331927f));
    p = fma(p, e, f2(-0.49999502f));
    p = fma(p, e, f2(1.f));
    float a, b;
    get(x, a, b);
    return fma(p, e, f2(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}
// Its derivative, from e.
__device__ __forceinline__ F2 softplus_slope(F2 x, F2 e) {
    float a, b, ea, eb, na, nb;
    get(x, a, b);
    get(e, ea, eb);
    get(add(e, f2(1.f)), na, nb);
    return mul(f2(rcp(na), rcp(nb)), f2(a >= 0.f ? 1.f : ea, b >= 0.f ? 1.f : eb));
}
__device__ __forceinline__ F2 sigmoid(F2 x) {
    float a, b;
    get(mul(x, f2(-1.4426950408889634f)), a, b);
    get(add(f2(ex2(a), ex2(b)), f2(1.f)), a, b);
    return f2(rcp(a), rcp(b));
}
template <int V>
__device__ __forceinline__ void softplus_all(float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = softplus(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            F2 e;
            get(softplus(f2(x[i], x[i + 1]), e), x[i], x[i + 1]);
        }
    }
}
template <int V>
__device__ __forceinline__ void sigmoid_all(float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = sigmoid(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) get(sigmoid(f2(x[i], x[i + 1])), x[i], x[i + 1]);
    }
}
// x becomes softplus(x), `slope` its derivative sigmoid(x).
template <int V>
__device__ __forceinline__ void softplus_slope_all(float (&x)[V], float (&slope)[V]) {
    if constexpr (V == 1) {
        const float e = exp_neg(x[0]), r = rcp(1.f + e);
        slope[0] = x[0] >= 0.f ? r : e * r;
        x[0] = softplus(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const F2 v = f2(x[i], x[i + 1]);
            F2 e;
            get(softplus(v, e), x[i], x[i + 1]);
            get(softplus_slope(v, e), slope[i], slope[i + 1]);
        }
    }
}
// s += x with what the sum's rounding leaves out kept in `rest`.
__device__ __forceinline__ void add_exactly(float& s, float& rest, float x) {
    const float t = __fadd_rn(s, x), z = __fsub_rn(t, s);
    rest = __fadd_rn(rest, __fadd_rn(__fsub_rn(s, __fsub_rn(t, z)), __fsub_rn(x, z)));
    s = t;
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
    alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) T x[V];
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
    // (the whole piece, aligned)
    __device__ __forceinline__ void load(const T* at) {
        constexpr int kB = V * (int)sizeof(T);
        using Word = typename std::conditional<kB >= 16, uint4, typename std::conditional<kB == 8, uint2, typename std::conditional<kB == 4, uint32_t, T>::type>::type>::type;
#pragma unroll
        for (int i = 0; i < kB / (int)sizeof(Word); ++i) reinterpret_cast<Word*>(x)[i] = reinterpret_cast<const Word*>(at)[i];
    }
    __device__ __forceinline__ void store(T* at) const {
        constexpr int kB = V * (int)sizeof(T);
        using Word = typename std::conditional<kB >= 16, uint4, typename std::conditional<kB == 8, uint2, typename std::conditional<kB == 4, uint32_t, T>::type>::type>::type;
#pragma unroll
        for (int i = 0; i < kB / (int)sizeof(Word); ++i) reinterpret_cast<Word*>(at)[i] = reinterpret_cast<const Word*>(x)[i];
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

// One such piece from global into shared memory, by the thread that reads it there: asynchronously where `vec` bytes allow it.
template <typename T, int V>
__device__ __forceinline__ void fetch(T* to, const T* from, int n, bool vec) {
    constexpr int kB = V * (int)sizeof(T);
    if constexpr (kB >= 4) {
        if (vec && n >= V) {
            const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
            if constexpr (kB >= 16) {
#pragma unroll
                for (int i = 0; i < kB; i += 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i), "l"(reinterpret_cast<const char*>(from) + i) : "memory");
            } else {
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(kB) : "memory");
            }
            return;
        }
    }
    Piece<T, V> x;
    x.load(from, n, vec);
    x.store(to, V, false);
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Places of channel c in a tile's row of pairs and of single values: 16-byte units, permuted so that the eight threads that
// stage a row, V channels each, write and read without bank conflicts (a thread's channels lie V apart from its neighbour's).
__device__ __forceinline__ int pair_at(int c) {
    const int u = c >> 1;
    return (u ^ ((u >> 3) & 3)) * 2 + (c & 1);
}
__device__ __forceinline__ int single_at(int c) {
    const int u = c >> 2;
    return (u ^ ((u >> 3) & 1)) * 4 + (c & 3);
}
template <int V>
__device__ __forceinline__ void put_pairs(float2* row, int c0, const float (&a)[V], const float (&b)[V]) {
    if constexpr (V == 1) {
        row[pair_at(c0)] = make_float2(a[0], b[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) *reinterpret_cast<float4*>(row + pair_at(c0 + i)) = make_float4(a[i], b[i], a[i + 1], b[i + 1]);
    }
}
template <int V>
__device__ __forceinline__ void get_pairs(const float2* row, int c0, float (&a)[V], float (&b)[V]) {
    if constexpr (V == 1) {
        const float2 x = row[pair_at(c0)];
        a[0] = x.x, b[0] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float4 x = *reinterpret_cast<const float4*>(row + pair_at(c0 + i));
            a[i] = x.x, b[i] = x.y, a[i + 1] = x.z, b[i + 1] = x.w;
        }
    }
}
template <int V>
__device__ __forceinline__ void put_singles(float* row, int c0, const float (&a)[V]) {
    if constexpr (V == 1) {
        row[single_at(c0)] = a[0];
    } else if constexpr (V == 2) {
        *reinterpret_cast<float2*>(row + single_at(c0)) = make_float2(a[0], a[1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(row + single_at(c0 + i)) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
    }
}
template <int V>
__device__ __forceinline__ void get_singles(const float* row, int c0, float (&a)[V]) {
    if constexpr (V == 1) {
        a[0] = row[single_at(c0)];
    } else if constexpr (V == 2) {
        const float2 x = *reinterpret_cast<const float2*>(row + single_at(c0));
        a[0] = x.x, a[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(row + single_at(c0 + i));
            a[i] = x.x, a[i + 1] = x.y, a[i + 2] = x.z, a[i + 3] = x.w;
        }
    }
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

// A tile's rows of B or C as float32, zeros on masked tokens, behind the last token and behind the N-th state: four
// neighbouring states of a token for each of the first (or every) 8 LPC x 32 / 8 threads.
template <typename T, int LPC>
struct States {
    static constexpr int kNp = 4 * LPC, kPieces = kSelTile * LPC, kPer = (kPieces + kSelThreads - 1) / kSelThreads;
    Piece<T, 4> x[kPer];
    __device__ __forceinline__ void load(const SelParams& p, const SelTensor& t, int b, int g, int l0, int l1) {
        const bool vec = t.vec >= 4 * (int)sizeof(T) && (t.sg * (int64_t)sizeof(T)) % (4 * sizeof(T)) == 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = threadIdx.x + i * kSelThreads, l = l0 + at / LPC, n = at % LPC * 4;
            x[i].zero();
            if ((kPieces % kSelThreads == 0 || at < kPieces) && n < p.N && l < l1 && live_at<T>(p, b, l))
                x[i].load(static_cast<const T*>(t.p) + b * t.sb + l * t.sl + g * t.sg + n, p.N - n, vec);
        }
    }
    // (each four with their places n ^ order)
    __device__ __forceinline__ void put(float* to, int order = 0) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = threadIdx.x + i * kSelThreads;
            if (kPieces % kSelThreads == 0 || at < kPieces)
                *reinterpret_cast<float4*>(to + 4 * at) = make_float4(to_f<T>(x[i].x[order]), to_f<T>(x[i].x[1 ^ order]), to_f<T>(x[i].x[2 ^ order]), to_f<T>(x[i].x[3 ^ order]));
        }
    }
};

}  // namespace sel
}  // namespace subq
