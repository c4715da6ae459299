// Root-mean-square norm over the last dimension of [rows, D] with the residual's addition, forward and backward:
//   r = x + res (in res's type),   xh = r rsqrt(mean(r^2) + eps),   y = xh w
//   g = dy w,   dr = rsqrt(..) (g - xh mean(g xh)) + dr_next,   dx = dres = dr,   dw = sum dy xh
// y is 16 or 32 bits wide, or e4m3 with a float32 scale for every 128 columns of a row:
//   scale = max(amax of y, 1e-30) / 448,   q = y / scale rounded to e4m3 (a NaN makes its scale and its 128 values NaN).
// The norm is of r as it is stored, so that the backward, which is given r, sees the same numbers.
//
// HBM-bound: a row is read once and written once. NW warps hold a row, 8 neighbouring columns K times a lane, in registers
// between the passes; 16 lanes have the 128 columns of a scale. The next row is on its way while one is worked on. The
// backward's CTAs stay for many rows with dw in registers: one partial row a CTA, summed by a second launch in a fixed order.
// 65536 x 768, bf16 with a float32 stream: forward 95 us (6.4 TB/s), backward 142 us (5.7 TB/s). 16384 x 1024 bf16 to 8 bits: 34 us
// (3.5 TB/s: latency; 14.7 warps an SM at 128 registers, issue slots 0.57 used).
#include <cuda_fp8.h>

#include "sel_common.cuh"

namespace subq {
namespace {

using sel::Piece;
using sel::need_vec;

constexpr int kSMs = 148;

template <int NW, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float (*red)[M], int warp_in_row, int group) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (NW > 1) {
        auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * NW) : "memory"); };
        sync();  // the sums before have been read
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < M; ++i) red[warp_in_row][i] = v[i];
        sync();
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int i = 0; i < M; ++i) v[i] += red[w][i];
    }
}

// The larger of two, a NaN where either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct Fp8 {};  // y in e4m3 with scales

// Is x within 8 float32 steps of the middle between two e4m3 neighbours (4 significant bits; below 2^-6, where their step
// no longer shrinks, one value in 10^5 of a block's range, it is not asked)? What float32 leaves of y / scale (four
// roundings) could lie on the other side of it.
__device__ __forceinline__ bool near_border(float x) { return (__float_as_uint(x) & 0xfffffu) - 0x7fff8u < 16u; }

// y / scale of such values again in float64, from r and w themselves: the rows' norm is the same on both sides of the
// quotient, so that q = 448 r w / max |r w|, exact but for two roundings of 2^-53. Rounded to float32 towards zero with the
// last bit set where anything was cut off, which the rounding to e4m3 that follows sees on the right side.
template <typename TR, int V>
__device__ __forceinline__ void exact_quotients(float (&f)[V], const Piece<TR, V>& r, const float* w, int c, int n, bool near) {
    double t[V], top = 0.;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        t[i] = i < n ? (double)to_f<TR>(r.x[i]) * (w ? (double)w[c + i] : 1.) : 0.;
        top = fmax(top, fabs(t[i]));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!near) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!near_border(f[i])) continue;
        const double q = 448. * t[i] / top;  // (the first product is exact: so is a value halfway between two)
        const float z = __double2float_rz(q);
        f[i] = (double)z == q ? z : __uint_as_float(__float_as_uint(z) | 1u);
    }
}

// A piece of a row: whole and aligned, or element by element.
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void rows_load(Piece<T, V>& x, const T* at, int n) {
    if constexpr (WHOLE) x.load(at);
    else x.load(at, n, false);
}
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void rows_store(const Piece<T, V>& x, T* at, int n) {
    if constexpr (WHOLE) {
        x.store(at);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) at[i] = x.x[i];
    }
}

// Weights of eight columns (1 without any, 0 behind the last column).
template <bool WHOLE, int V>
__device__ __forceinline__ void weights(const RmsNormParams& p, int c, int n, float (&w)[V]) {
    if (!p.w) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 1.f;
    } else if (WHOLE) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 x = n > 0 ? *reinterpret_cast<const float4*>(p.w + c + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = i < n ? p.w[c + i] : 0.f;
    }
}

// A CTA of kWarps warps works on kWarps / NW rows at once.
template <int NW>
struct Rows {
    static constexpr int kWarps = NW > 4 ? NW : 4, kGroups = kWarps / NW, kThreads = 32 * kWarps;
};

template <typename TX, typename TR, typename TY, int K, int NW, bool WHOLE>
__global__ void __launch_bounds__(Rows<NW>::kThreads, NW <= 4 ? 4 : 1) rms_fwd_kernel(const RmsNormParams p) {
    constexpr int V = 8;
    __shared__ float red[Rows<NW>::kGroups][NW][1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / NW, in_row = warp % NW;
    const int c0 = (in_row * 32 + lane) * V;
    constexpr int kStep = NW * 32 * V;
    const int64_t step = (int64_t)gridDim.x * Rows<NW>::kGroups;
    Piece<TX, V> nx[K];
    Piece<TR, V> nr[K];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = c0 + k * kStep, n = p.D - c;
            nx[k].zero();
            nr[k].zero();
            if (n > 0) {
                rows_load<WHOLE>(nx[k], static_cast<const TX*>(p.x) + row * p.x_s + c, n);
                if (p.res) rows_load<WHOLE>(nr[k], static_cast<const TR*>(p.res) + row * p.res_s + c, n);
            }
        }
    };
    int64_t row = (int64_t)blockIdx.x * Rows<NW>::kGroups + group;
    if (row < p.rows) load(row);
    for (; row < p.rows; row += step) {
        float f[K][V];  // r, then y, then y / scale
        Piece<TR, V> r[K];
        float ss[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = c0 + k * kStep, n = p.D - c;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                f[k][i] = to_f<TX>(nx[k].x[i]);
                if (p.res) f[k][i] += to_f<TR>(nr[k].x[i]);
                r[k].x[i] = from_f<TR>(f[k][i]);  // (without a residual a copy: TR holds x)
                f[k][i] = to_f<TR>(r[k].x[i]);
                ss[0] = fmaf(f[k][i], f[k][i], ss[0]);
            }
            if (p.r && n > 0) rows_store<WHOLE>(r[k], static_cast<TR*>(p.r) + row * p.r_s + c, n);
        }
        if (row + step < p.rows) load(row + step);
        float rms = 1.f;
        if (p.norm) {
            row_sums<NW, 1>(ss, red[group], in_row, group);
            rms = 1.f / sqrtf(ss[0] / (float)p.D + p.eps);
        }
        if constexpr (std::is_same<TY, Fp8>::value) {
            float top[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = c0 + k * kStep, n = p.D - c;
                float w[V];
                weights<WHOLE>(p, c, n, w);
                top[k] = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    f[k][i] = f[k][i] * rms * w[i];
                    top[k] = max_nan(top[k], i < n ? fabsf(f[k][i]) : 0.f);
                }
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < K; ++k) top[k] = max_nan(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
            bool near[K], any = false;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = c0 + k * kStep, n = p.D - c;
                const float inv = __fdiv_rn(448.f, max_nan(top[k], 1e-30f));
                near[k] = false;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    f[k][i] *= inv;
                    near[k] |= near_border(f[k][i]);
                }
                near[k] = near[k] && top[k] > 1e-30f && top[k] < INFINITY && n > 0;
                any |= near[k];
            }
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (__any_sync(0xffffffffu, near[k])) exact_quotients<TR, V>(f[k], r[k], p.w, c0 + k * kStep, p.D - c0 - k * kStep, near[k]);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = c0 + k * kStep, n = p.D - c;
                if (n <= 0) continue;
                if ((lane & 15) == 0) p.scale[row * p.scale_s + c / 128] = __fdiv_rn(max_nan(top[k], 1e-30f), 448.f);
                Piece<uint8_t, V> q;
#pragma unroll
                for (int i = 0; i < V; i += 2)
                    reinterpret_cast<__nv_fp8x2_storage_t*>(q.x)[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(f[k][i], f[k][i + 1]), __NV_SATFINITE, __NV_E4M3);
                rows_store<WHOLE>(q, static_cast<uint8_t*>(p.y) + row * p.y_s + c, n);
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = c0 + k * kStep, n = p.D - c;
                if (n <= 0) continue;
                float w[V];
                weights<WHOLE>(p, c, n, w);
                Piece<TY, V> y;
#pragma unroll
                for (int i = 0; i < V; ++i) y.x[i] = from_f<TY>(f[k][i] * rms * w[i]);
                rows_store<WHOLE>(y, static_cast<TY*>(p.y) + row * p.y_s + c, n);
            }
        }
    }
}

// TY: type of dy (and of dx, where it is not TR).
template <typename TX, typename TR, typename TY, int K, int NW, bool WHOLE>
__global__ void __launch_bounds__(Rows<NW>::kThreads) rms_bwd_kernel(const RmsNormParams p) {
    constexpr int V = 8;
    __shared__ float red[Rows<NW>::kGroups][NW][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / NW, in_row = warp % NW;
    const int c0 = (in_row * 32 + lane) * V;
    constexpr int kStep = NW * 32 * V;
    const int64_t step = (int64_t)gridDim.x * Rows<NW>::kGroups;
    float dw[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * Rows<NW>::kGroups + group; row < p.rows; row += step) {
        Piece<TY, V> dy[K];
        Piece<TR, V> r[K], dn[K];
        float sums[2] = {0.f, 0.f};  // r^2, dy w r
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = c0 + k * kStep, n = p.D - c;
            dy[k].zero();
            r[k].zero();
            dn[k].zero();
            if (n > 0) {
                rows_load<WHOLE>(r[k], static_cast<const TR*>(p.r) + row * p.r_s + c, n);
                rows_load<WHOLE>(dy[k], static_cast<const TY*>(p.dy) + row * p.dy_s + c, n);
                if (p.dr) rows_load<WHOLE>(dn[k], static_cast<const TR*>(p.dr) + row * p.dr_s + c, n);
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float w[V];
            weights<WHOLE>(p, c0 + k * kStep, p.D - c0 - k * kStep, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float rf = to_f<TR>(r[k].x[i]);
                sums[0] = fmaf(rf, rf, sums[0]);
                sums[1] = fmaf(to_f<TY>(dy[k].x[i]) * w[i], rf, sums[1]);
            }
        }
        row_sums<NW, 2>(sums, red[group], in_row, group);
        const float rms = 1.f / sqrtf(sums[0] / (float)p.D + p.eps), m = rms * (sums[1] / (float)p.D);  // mean(g xh)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = c0 + k * kStep, n = p.D - c;
            Piece<TX, V> ox;
            Piece<TR, V> ores;
            float w[V];
            weights<WHOLE>(p, c, n, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = to_f<TR>(r[k].x[i]) * rms, g = to_f<TY>(dy[k].x[i]);
                dw[k][i] = fmaf(g, xh, dw[k][i]);
                const float d = fmaf(rms, fmaf(-xh, m, g * w[i]), to_f<TR>(dn[k].x[i]));
                ox.x[i] = from_f<TX>(d);
                ores.x[i] = from_f<TR>(d);
            }
            if (n > 0) {
                if (p.dx) rows_store<WHOLE>(ox, static_cast<TX*>(p.dx) + row * p.dx_s + c, n);
                if (p.dres) rows_store<WHOLE>(ores, static_cast<TR*>(p.dres) + row * p.dres_s + c, n);
            }
        }
    }
    if (!p.part) return;
    // the CTA's groups one after another, in a fixed order
    float* part = p.part + (int64_t)blockIdx.x * p.D;
    for (int g = 0; g < Rows<NW>::kGroups; ++g) {
        if (group == g)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = c0 + k * kStep + i;
                    if (c < p.D) part[c] = g ? part[c] + dw[k][i] : dw[k][i];
                }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) rms_dw_kernel(const float* part, float* dw, int D, int parts) {
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), sub = threadIdx.x >> 5;
    float s = 0.f;
    if (c < D)
#pragma unroll 8
        for (int k = sub; k < parts; k += 8) s += part[(int64_t)k * D + c];
    __shared__ float red[8][32];
    red[sub][threadIdx.x & 31] = s;
    __syncthreads();
    if (sub || c >= D) return;
    s = 0.f;
    for (int k = 0; k < 8; ++k) s += red[k][threadIdx.x];
    dw[c] = s;
}

int es(int dtype) { return dtype == SUBQ_FP32 ? 4 : 2; }
// Do rows of `size`-byte elements allow whole pieces of 8 (or are there none)?
bool rows_fit(const void* at, int64_t stride, int size) {
    const int need = size == 1 ? 8 : 16;
    return !at || (reinterpret_cast<uintptr_t>(at) % need == 0 && stride * size % need == 0);
}
bool whole(const RmsNormParams& p) { return p.D % 8 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0; }

template <typename F>
cudaError_t by_width(int D, F f) {
    auto run = [&](auto k, auto nw) { return f(k, nw); };
    using std::integral_constant;
    if (D <= 256) return run(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (D <= 512) return run(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    if (D <= 768) return run(integral_constant<int, 3>{}, integral_constant<int, 1>{});
    if (D <= 1024) return run(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (D <= 2048) return run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    if (D <= 4096) return run(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    if (D <= 8192) return run(integral_constant<int, 4>{}, integral_constant<int, 8>{});
    return run(integral_constant<int, 4>{}, integral_constant<int, 16>{});
}

template <typename TX, typename TR, typename TY>
cudaError_t fwd_typed(const RmsNormParams& p, cudaStream_t st) {
    const bool all = whole(p) && rows_fit(p.x, p.x_s, sizeof(TX)) && rows_fit(p.res, p.res_s, sizeof(TR)) && rows_fit(p.r, p.r_s, sizeof(TR)) && rows_fit(p.y, p.y_s, sizeof(TY));
    return by_width(p.D, [&](auto k, auto nw) {
        constexpr int K = decltype(k)::value, NW = decltype(nw)::value;
        const int64_t most = (int64_t)kSMs * (2048 / Rows<NW>::kThreads), need = (p.rows + Rows<NW>::kGroups - 1) / Rows<NW>::kGroups;
        const unsigned blocks = (unsigned)(need < most ? need : most);
        if (all) rms_fwd_kernel<TX, TR, TY, K, NW, true><<<blocks, Rows<NW>::kThreads, 0, st>>>(p);
        else rms_fwd_kernel<TX, TR, TY, K, NW, false><<<blocks, Rows<NW>::kThreads, 0, st>>>(p);
        return cudaGetLastError();
    });
}

template <typename TX, typename TR>
cudaError_t bwd_typed(const RmsNormParams& p, cudaStream_t st, int* launches) {
    using TY = TX;
    const bool all = whole(p) && rows_fit(p.dy, p.dy_s, sizeof(TY)) && rows_fit(p.r, p.r_s, sizeof(TR)) && rows_fit(p.dr, p.dr_s, sizeof(TR)) && rows_fit(p.dx, p.dx_s, sizeof(TX)) &&
                     rows_fit(p.dres, p.dres_s, sizeof(TR));
    return by_width(p.D, [&](auto k, auto nw) {
        constexpr int K = decltype(k)::value, NW = decltype(nw)::value;
        const int64_t most = NW >= 8 ? kSMs : kRmsParts, need = (p.rows + Rows<NW>::kGroups - 1) / Rows<NW>::kGroups;
        const int blocks = (int)(need < most ? need : most);
        if (all) rms_bwd_kernel<TX, TR, TY, K, NW, true><<<blocks, Rows<NW>::kThreads, 0, st>>>(p);
        else rms_bwd_kernel<TX, TR, TY, K, NW, false><<<blocks, Rows<NW>::kThreads, 0, st>>>(p);
        *launches = 1;
        if (p.part) {
            rms_dw_kernel<<<(p.D + 31) / 32, 256, 0, st>>>(p.part, p.dw, p.D, blocks);
            *launches = 2;
        }
        return cudaGetLastError();
    });
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormParams& p, int x, int r, int y, cudaStream_t st) {
    using b = __nv_bfloat16;
    using h = __half;
    if (x == SUBQ_FP32)
        return y == SUBQ_FP32 ? fwd_typed<float, float, float>(p, st) : y == SUBQ_FP16 ? fwd_typed<float, float, h>(p, st)
               : y == SUBQ_BF16 ? fwd_typed<float, float, b>(p, st) : fwd_typed<float, float, Fp8>(p, st);
    if (x == SUBQ_FP16) {
        if (r == SUBQ_FP32) return y < 0 ? fwd_typed<h, float, Fp8>(p, st) : fwd_typed<h, float, h>(p, st);
        return y < 0 ? fwd_typed<h, h, Fp8>(p, st) : fwd_typed<h, h, h>(p, st);
    }
    if (r == SUBQ_FP32) return y < 0 ? fwd_typed<b, float, Fp8>(p, st) : fwd_typed<b, float, b>(p, st);
    return y < 0 ? fwd_typed<b, b, Fp8>(p, st) : fwd_typed<b, b, b>(p, st);
}

cudaError_t launch_rms_norm_bwd(const RmsNormParams& p, int x, int r, cudaStream_t st, int* launches) {
    using b = __nv_bfloat16;
    using h = __half;
    if (x == SUBQ_FP32) return bwd_typed<float, float>(p, st, launches);
    if (x == SUBQ_FP16) return r == SUBQ_FP32 ? bwd_typed<h, float>(p, st, launches) : bwd_typed<h, h>(p, st, launches);
    return r == SUBQ_FP32 ? bwd_typed<b, float>(p, st, launches) : bwd_typed<b, b>(p, st, launches);
}

}  // namespace subq
