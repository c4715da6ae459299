// Selective scan, forward: one CTA of 256 threads walks 256 / LPC channels of one sequence (or of one of its segments)
// through tiles of 32 tokens. A tile's u and dt come in as whole rows, dt = softplus(raw + bias) and dt u are formed once
// per token and channel and left in shared memory, the states stay in registers, and y goes back through shared memory to
// the threads that hold u and z for the output. The next tile is on its way meanwhile.
//
// Bound by instruction issue and the exponential unit (one exponential and about nine packed or single operations a
// state), not by memory. Few channels: the sequence is cut into segments; a first launch finds what each leaves of a zero
// state and the sum of its step sizes (a segment's decay is exp(A sum dt)), and the walk's CTAs chain those before theirs.
#pragma once

#include "sel_common.cuh"

namespace subq {
namespace sel {

// State at the begin of segment `seg`: what the segments before it make of S_in.
template <int LPC>
__device__ __forceinline__ void chain_in(const SelParams& p, int seg, int b, int d, int q, const float (&A2)[4], float (&h)[4]) {
    constexpr int kNp = 4 * LPC;
    for (int s = 0; s < seg; ++s) {
        const int64_t at = ((int64_t)s * p.B + b) * p.D + d;
        const float4 x = *reinterpret_cast<const float4*>(p.seg_h + at * kNp + 4 * q);
        const float dt = p.seg_dt[at];
        h[0] = fmaf(decay(A2[0] * dt), h[0], h[0]) + x.x;
        h[1] = fmaf(decay(A2[1] * dt), h[1], h[1]) + x.y;
        h[2] = fmaf(decay(A2[2] * dt), h[2], h[2]) + x.z;
        h[3] = fmaf(decay(A2[3] * dt), h[3], h[3]) + x.w;
    }
}

constexpr float kLog2e = 1.4426950408889634f;

template <int LPC>
__device__ __forceinline__ void load_A(const SelParams& p, int d, bool in, int q, float (&A2)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] = in && 4 * q + i < p.N ? p.A[(int64_t)d * p.N + 4 * q + i] * kLog2e : 0.f;
}

template <typename T, int LPC, bool WALK>
__global__ void __launch_bounds__(kSelThreads, LPC <= 8 ? 3 : 2) sel_fwd_kernel(const SelParams p) {
    using P = Place<T, LPC>;
    constexpr int kNp = 4 * LPC, V = P::kV, kCh = P::kCh;
    extern __shared__ __align__(16) unsigned char smem[];
    float2* sdt = reinterpret_cast<float2*>(smem);                      // [tile][channels]: dt, dt u
    float* sB = reinterpret_cast<float*>(sdt + kSelTile * kCh);         // [tile][states]
    float* sC = sB + kSelTile * kNp;
    float* sy = sC + kSelTile * kNp;                                    // [tile][channels]
    const P at(p);
    const int seg = blockIdx.y, first = seg * p.seg_tokens, last = min(p.L, first + p.seg_tokens);
    const int lane = threadIdx.x & 31, q = lane & (LPC - 1), ch = threadIdx.x / LPC, d = at.d0 + ch;
    const bool in = ch < at.nch;
    float A2[4], h0[4] = {0.f, 0.f, 0.f, 0.f};
    load_A<LPC>(p, d, in, q, A2);
    const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
    if (WALK && in) {
        if (p.S_in)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) h0[i] = p.S_in[((int64_t)at.b * p.D + d) * p.N + 4 * q + i];
        chain_in<LPC>(p, seg, at.b, d, q, A2, h0);
    }
    F2 h01 = f2(h0[0], h0[1]), h23 = f2(h0[2], h0[3]);
    float bias[V], Dw[V], dt_sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool has = i < at.left;
        bias[i] = has && p.dt_bias ? p.dt_bias[at.d0 + at.c0 + i] : 0.f;
        Dw[i] = WALK && has && p.Dw ? p.Dw[at.d0 + at.c0 + i] : 0.f;
        dt_sum[i] = 0.f;
    }
    constexpr int kBytes = need_vec<V * (int)sizeof(T)>();
    const bool even = at.d0 % V == 0;
    const bool vu = even && p.u.vec >= kBytes, vd = even && p.dt.vec >= kBytes, vz = even && p.z.vec >= kBytes, vo = even && p.out.vec >= kBytes;
    const bool outs = WALK && p.out.p;
    Piece<T, V> u, dt, z;
    States<T, LPC> Bs, Cs;
    auto load = [&](int l0) {
        const int l = l0 + at.row;
        const bool live = l < last && live_at<T>(p, at.b, l);
        u.zero(); dt.zero(); z.zero();
        if (live) {
            u.load(row_of<T>(p.u, at.b, l, at.d0 + at.c0), at.left, vu);
            dt.load(row_of<T>(p.dt, at.b, l, at.d0 + at.c0), at.left, vd);
            if (outs && p.z.p) z.load(row_of<T>(p.z, at.b, l, at.d0 + at.c0), at.left, vz);
        }
        Bs.load(p, p.Bm, at.b, at.g, l0, last);
        if (outs) Cs.load(p, p.C, at.b, at.g, l0, last);
        return live;
    };
    bool live = load(first);
    for (int l0 = first; l0 < last; l0 += kSelTile) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = to_f<T>(dt.x[i]) + bias[i];
            if (p.softplus) s = softplus(s);
            if (!live || i >= at.left) s = 0.f;
            if (!WALK) dt_sum[i] += s;
            sdt[at.row * kCh + at.c0 + i] = make_float2(s, s * to_f<T>(u.x[i]));
        }
        Bs.put(sB);
        if (outs) Cs.put(sC);
        const Piece<T, V> u_now = u, z_now = z;
        const bool live_now = live;
        if (l0 + kSelTile < last) live = load(l0 + kSelTile);
        __syncthreads();
#pragma unroll 2
        for (int t4 = 0; t4 < kSelTile; t4 += 4) {
            if (WALK && p.kept && t4 % kSelKeep == 0 && in && l0 + t4 < p.L) {
                float4 x;
                get(h01, x.x, x.y);
                get(h23, x.z, x.w);
                *reinterpret_cast<float4*>(p.kept + (((int64_t)at.b * ((p.L + kSelKeep - 1) / kSelKeep) + (l0 + t4) / kSelKeep) * p.D + d) * kNp + 4 * q) = x;
            }
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t4 + i;
                const float2 s = sdt[t * kCh + ch];
                const float4 Bv = *reinterpret_cast<const float4*>(sB + t * kNp + 4 * q);
                const F2 dt2 = f2(s.x), du2 = f2(s.y);
                const F2 e01 = decay(mul(dt2, A01)), e23 = decay(mul(dt2, A23));
                h01 = add(h01, fma(e01, h01, mul(du2, f2(Bv.x, Bv.y))));
                h23 = add(h23, fma(e23, h23, mul(du2, f2(Bv.z, Bv.w))));
                if (outs) {
                    const float4 Cv = *reinterpret_cast<const float4*>(sC + t * kNp + 4 * q);
                    y[i] = both(fma(h23, f2(Cv.z, Cv.w), mul(h01, f2(Cv.x, Cv.y))));
                }
            }
            if (outs) {
                const float s = lane_sums4<LPC>(y, lane);
                if (q < 4) sy[(t4 + q) * kCh + ch] = s;
            }
        }
        __syncthreads();
        if (outs && l0 + at.row < last && at.left > 0) {
            Piece<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float y = fmaf(Dw[i], to_f<T>(u_now.x[i]), sy[at.row * kCh + at.c0 + i]);
                if (p.z.p) {
                    const float zf = to_f<T>(z_now.x[i]);
                    y *= zf * sigmoid(zf);
                }
                o.x[i] = from_f<T>(live_now ? y : 0.f);
            }
            o.store(const_cast<T*>(row_of<T>(p.out, at.b, l0 + at.row, at.d0 + at.c0)), at.left, vo);
        }
    }
    float h[4];
    get(h01, h[0], h[1]);
    get(h23, h[2], h[3]);
    if (WALK) {
        if (p.S_out && last == p.L && in)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) p.S_out[((int64_t)at.b * p.D + d) * p.N + 4 * q + i] = h[i];
        return;
    }
    const int64_t to = ((int64_t)seg * p.B + at.b) * p.D;
    if (in) *reinterpret_cast<float4*>(p.seg_h + (to + d) * kNp + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
    __syncthreads();  // sum of the rows' step sizes, in a fixed order
#pragma unroll
    for (int i = 0; i < V; ++i) sy[at.row * kCh + at.c0 + i] = dt_sum[i];
    __syncthreads();
    if (threadIdx.x < at.nch) {
        float s = 0.f;
        for (int r = 0; r < kSelTile; ++r) s += sy[r * kCh + threadIdx.x];
        p.seg_dt[to + at.d0 + threadIdx.x] = s;
    }
}

// Token by token, without shared memory: a lane has four states of a channel and reads its token's values by itself. For
// single tokens (the states' 8 N D bytes a sequence, or the launch) and calls of a few.
template <typename T, int LPC>
__global__ void __launch_bounds__(kSelThreads) sel_step_kernel(const SelParams p) {
    const int q = threadIdx.x & (LPC - 1);
    const int64_t channel = ((int64_t)blockIdx.x * kSelThreads + threadIdx.x) / LPC;
    const bool in = channel < (int64_t)p.B * p.D;
    const int b = in ? (int)(channel / p.D) : 0, d = in ? (int)(channel - (int64_t)b * p.D) : 0, g = d / p.Dg;
    const bool whole = p.N % 4 == 0;  // 16-byte accesses of the states (their base is aligned to 16 bytes, or N is not used so)
    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t sat = ((int64_t)b * p.D + d) * p.N + 4 * q;
    const bool vec = whole && ((reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.S_out) | reinterpret_cast<uintptr_t>(p.A)) & 15) == 0;
    if (vec) {
        const bool has = in && 4 * q < p.N;
        const float4 a = has ? *reinterpret_cast<const float4*>(p.A + (int64_t)d * p.N + 4 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 x = has && p.S_in ? *reinterpret_cast<const float4*>(p.S_in + sat) : make_float4(0.f, 0.f, 0.f, 0.f);
        A2[0] = a.x * kLog2e; A2[1] = a.y * kLog2e; A2[2] = a.z * kLog2e; A2[3] = a.w * kLog2e;
        h[0] = x.x; h[1] = x.y; h[2] = x.z; h[3] = x.w;
    } else {
        load_A<LPC>(p, d, in, q, A2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && p.S_in && 4 * q + i < p.N) h[i] = p.S_in[sat + i];
    }
    const float bias = in && p.dt_bias ? p.dt_bias[d] : 0.f, Dw = in && p.Dw ? p.Dw[d] : 0.f;
    for (int l = 0; l < p.L; ++l) {
        const bool live = in && live_at<T>(p, b, l);
        float y = 0.f, u = 0.f, z = 0.f;
        if (live) {
            u = to_f<T>(*row_of<T>(p.u, b, l, d));
            float dt = to_f<T>(*row_of<T>(p.dt, b, l, d)) + bias;
            if (p.z.p) z = to_f<T>(*row_of<T>(p.z, b, l, d));
            const T* Bp = row_of<T>(p.Bm, b, l, 0) + g * p.Bm.sg + 4 * q;
            const T* Cp = row_of<T>(p.C, b, l, 0) + g * p.C.sg + 4 * q;
            float Bv[4], Cv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool has = 4 * q + i < p.N;
                Bv[i] = has ? to_f<T>(Bp[i]) : 0.f;
                Cv[i] = has ? to_f<T>(Cp[i]) : 0.f;
            }
            if (p.softplus) dt = softplus(dt);
            const float du = dt * u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] += fmaf(decay(dt * A2[i]), h[i], du * Bv[i]);
                y = fmaf(Cv[i], h[i], y);
            }
        }
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (in && q == 0 && p.out.p) {
            y = fmaf(Dw, u, y);
            if (p.z.p) y *= z * sigmoid(z);
            *const_cast<T*>(row_of<T>(p.out, b, l, d)) = from_f<T>(live ? y : 0.f);
        }
    }
    if (in && p.S_out) {
        if (vec) {
            if (4 * q < p.N) *reinterpret_cast<float4*>(p.S_out + sat) = make_float4(h[0], h[1], h[2], h[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) p.S_out[sat + i] = h[i];
        }
    }
}

template <int LPC>
constexpr size_t fwd_smem() {
    return (size_t)kSelTile * (kSelThreads / LPC) * 12 + (size_t)kSelTile * 4 * LPC * 8;
}

template <typename T, int LPC, bool WALK>
cudaError_t launch_fwd_kernel(const SelParams& p, cudaStream_t st) {
    constexpr size_t smem = fwd_smem<LPC>();
    if (smem > 48 * 1024) {
        cudaError_t err = cudaFuncSetAttribute(sel_fwd_kernel<T, LPC, WALK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
    }
    const int kCh = kSelThreads / LPC;
    const dim3 grid((unsigned)(p.B * p.G * ((p.Dg + kCh - 1) / kCh)), (unsigned)(WALK ? p.nseg : p.nseg - 1));
    sel_fwd_kernel<T, LPC, WALK><<<grid, kSelThreads, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_fwd(const SelParams& p, SelPass pass, cudaStream_t st) {
    auto run = [&](auto lpc) {
        constexpr int LPC = decltype(lpc)::value;
        return pass == kSelWalk ? launch_fwd_kernel<T, LPC, true>(p, st) : launch_fwd_kernel<T, LPC, false>(p, st);
    };
    switch (sel_lanes(p.N)) {
        case 4: return run(std::integral_constant<int, 4>{});
        case 8: return run(std::integral_constant<int, 8>{});
        case 16: return run(std::integral_constant<int, 16>{});
        default: return run(std::integral_constant<int, 32>{});
    }
}

template <typename T>
cudaError_t launch_step(const SelParams& p, cudaStream_t st) {
    auto run = [&](auto lpc) {
        constexpr int LPC = decltype(lpc)::value;
        const int64_t threads = (int64_t)p.B * p.D * LPC;
        sel_step_kernel<T, LPC><<<(unsigned)((threads + kSelThreads - 1) / kSelThreads), kSelThreads, 0, st>>>(p);
        return cudaGetLastError();
    };
    switch (sel_lanes(p.N)) {
        case 4: return run(std::integral_constant<int, 4>{});
        case 8: return run(std::integral_constant<int, 8>{});
        case 16: return run(std::integral_constant<int, 16>{});
        default: return run(std::integral_constant<int, 32>{});
    }
}

}  // namespace sel
}  // namespace subq
