// Selective scan, forward: one CTA of 256 threads walks 256 / LPC channels of one sequence (or of one of its segments)
// through tiles of 32 tokens. A tile's u and dt come in as whole rows, dt = softplus(raw + bias) and dt u are formed once
// per token and channel and left in shared memory, the states stay in registers, and y goes back through shared memory to
// the threads that hold u and z for the output. The next tile is on its way meanwhile.
//
// Bound by instruction issue and the FMA pipe (a state and token take one exponential, nine multiply-adds, two states at a
// time, and three selections), not by memory: 65536 x 1536 channels of 16 states take 1529 us, a third of them the
// segments; 124 us would be its bytes, 360 us its exponentials alone. Few channels: the sequence is cut into segments; a first launch finds what each leaves of a zero
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
        h[0] = decayed(A2[0] * dt, h[0]) + x.x;
        h[1] = decayed(A2[1] * dt, h[1]) + x.y;
        h[2] = decayed(A2[2] * dt, h[2]) + x.z;
        h[3] = decayed(A2[3] * dt, h[3]) + x.w;
    }
}

constexpr float kLog2e = 1.4426950408889634f;

template <int LPC>
__device__ __forceinline__ void load_A(const SelParams& p, int d, bool in, int q, float (&A2)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] = in && 4 * q + i < p.N ? p.A[(int64_t)d * p.N + 4 * q + i] * kLog2e : 0.f;
}

template <typename T, int LPC, bool OUTS>
__global__ void __launch_bounds__(kSelThreads, LPC <= 8 ? kSelResident : 2) sel_fwd_kernel(const SelParams p) {
    using P = Place<T, LPC>;
    constexpr int kNp = 4 * LPC, V = P::kV, kCh = P::kCh;
    extern __shared__ __align__(16) unsigned char smem[];
    float2* sdt = reinterpret_cast<float2*>(smem);                      // [tile][channels]: dt, dt u; then y
    float* sB = reinterpret_cast<float*>(sdt + kSelTile * kCh);         // [tile][states]
    float* sC = sB + kSelTile * kNp;
    float* sbias = sC + kSelTile * kNp;                                 // [channels]: dt_bias, D
    float* sD = sbias + kCh;
    T* raw = reinterpret_cast<T*>(sD + kCh) + threadIdx.x * V;          // two turns of u, dt, z: a thread's own pieces
    constexpr int kRaw = kSelTile * kCh;
    const P at(p);
    const int seg = blockIdx.y, first = seg * p.seg_tokens, last = min(p.L, first + p.seg_tokens);
    const int lane = threadIdx.x & 31, q = lane & (LPC - 1), ch = threadIdx.x / LPC, cp = pair_at(ch), d = at.d0 + ch;
    const bool in = ch < at.nch;
    constexpr int kBytes = need_vec<V * (int)sizeof(T)>();
    const bool even = at.d0 % V == 0;
    const bool vu = even && p.u.vec >= kBytes, vd = even && p.dt.vec >= kBytes, vz = even && p.z.vec >= kBytes, vo = even && p.out.vec >= kBytes;
    constexpr bool outs = OUTS;
    States<T, LPC> Bs, Cs;
    auto load = [&](int l0, int turn) {
        const int l = l0 + at.row;
        if (l < last && at.left > 0) {  // (a masked token's piece is fetched, but not used)
            T* to = raw + turn * 3 * kRaw;
            fetch<T, V>(to, row_of<T>(p.u, at.b, l, at.d0 + at.c0), at.left, vu);
            fetch<T, V>(to + kRaw, row_of<T>(p.dt, at.b, l, at.d0 + at.c0), at.left, vd);
            if (outs && p.z.p) fetch<T, V>(to + 2 * kRaw, row_of<T>(p.z, at.b, l, at.d0 + at.c0), at.left, vz);
        }
        fetch_commit();
        Bs.load(p, p.Bm, at.b, at.g, l0, last);
        if (outs) Cs.load(p, p.C, at.b, at.g, l0, last);
    };
    load(first, 0);
    for (int i = threadIdx.x; i < kCh; i += kSelThreads) {
        sbias[i] = i < at.nch && p.dt_bias ? p.dt_bias[at.d0 + i] : 0.f;
        sD[i] = outs && i < at.nch && p.Dw ? p.Dw[at.d0 + i] : 0.f;
    }
    float A2[4], h0[4] = {0.f, 0.f, 0.f, 0.f};
    load_A<LPC>(p, d, in, q, A2);
    const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
    if (in) {
        if (p.S_in)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) h0[i] = p.S_in[((int64_t)at.b * p.D + d) * p.N + 4 * q + i];
        chain_in<LPC>(p, seg, at.b, d, q, A2, h0);
    }
    F2 h01 = f2(h0[0], h0[1]), h23 = f2(h0[2], h0[3]);
    __syncthreads();
    int turn = 0;
    for (int l0 = first; l0 < last; l0 += kSelTile, turn ^= 1) {
        const bool live = l0 + at.row < last && live_at<T>(p, at.b, l0 + at.row);
        const T* mine = raw + turn * 3 * kRaw;
        fetch_wait<0>();
        {
            Piece<T, V> u, dt;
            u.load(mine, V, true);
            dt.load(mine + kRaw, V, true);
            float s[V];
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] = to_f<T>(dt.x[i]) + sbias[at.c0 + i];
            if (p.softplus) softplus_all(s);
            float su[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool has = live && i < at.left;
                su[i] = has ? s[i] * to_f<T>(u.x[i]) : 0.f;
                s[i] = has ? s[i] : 0.f;
            }
            put_pairs(sdt + at.row * kCh, at.c0, s, su);
        }
        Bs.put(sB);
        if (outs) Cs.put(sC);
        if (l0 + kSelTile < last) load(l0 + kSelTile, turn ^ 1);
        __syncthreads();
#pragma unroll 2
        for (int t4 = 0; t4 < kSelTile; t4 += 4) {
            if (p.kept && t4 % kSelKeep == 0 && in && l0 + t4 < p.L) {
                float4 x;
                get(h01, x.x, x.y);
                get(h23, x.z, x.w);
                *reinterpret_cast<float4*>(p.kept + (((int64_t)at.b * ((p.L + kSelKeep - 1) / kSelKeep) + (l0 + t4) / kSelKeep) * p.D + d) * kNp + 4 * q) = x;
            }
            Factor f01[4], f23[4];  // what does not wait for the state, for four tokens
            float du[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 s = sdt[(t4 + i) * kCh + cp];
                f01[i] = factor(mul(f2(s.x), A01));
                f23[i] = factor(mul(f2(s.x), A23));
                du[i] = s.y;
            }
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 Bv = *reinterpret_cast<const float4*>(sB + (t4 + i) * kNp + 4 * q);
                h01 = fma(f2(du[i]), f2(Bv.x, Bv.y), decayed(f01[i], h01));
                h23 = fma(f2(du[i]), f2(Bv.z, Bv.w), decayed(f23[i], h23));
                if (outs) {
                    const float4 Cv = *reinterpret_cast<const float4*>(sC + (t4 + i) * kNp + 4 * q);
                    y[i] = both(fma(h23, f2(Cv.z, Cv.w), mul(h01, f2(Cv.x, Cv.y))));
                }
            }
            if (outs) {
                const float s = lane_sums4<LPC>(y, lane);
                if (q < 4) sdt[(t4 + q) * kCh + cp].x = s;  // (the channel's lanes have read these tokens: the sum is of all of them)
            }
        }
        __syncthreads();
        if (outs && l0 + at.row < last && at.left > 0) {
            Piece<T, V> u, z, o;
            u.load(mine, V, true);
            float gate[V], ys[V], unused[V];
            get_pairs(sdt + at.row * kCh, at.c0, ys, unused);
            if (p.z.p) {
                z.load(mine + 2 * kRaw, V, true);
#pragma unroll
                for (int i = 0; i < V; ++i) gate[i] = to_f<T>(z.x[i]);
                sigmoid_all(gate);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float y = fmaf(sD[at.c0 + i], to_f<T>(u.x[i]), ys[i]);
                if (p.z.p) y *= to_f<T>(z.x[i]) * gate[i];
                o.x[i] = from_f<T>(live ? y : 0.f);
            }
            o.store(const_cast<T*>(row_of<T>(p.out, at.b, l0 + at.row, at.d0 + at.c0)), at.left, vo);
        }
    }
    float h[4];
    get(h01, h[0], h[1]);
    get(h23, h[2], h[3]);
    if (p.S_out && last == p.L && in)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * q + i < p.N) p.S_out[((int64_t)at.b * p.D + d) * p.N + 4 * q + i] = h[i];
}

// What a segment leaves of a zero state, and the sum of its step sizes (BACK: what it hands of a zero adjoint to the segment
// before it). Not a recurrence but a sum, h = sum_t exp(A (dt_{t+1} + .. + dt_last)) dt_t u_t B_t (BACK: P = sum_t exp(A (dt_first
// + .. + dt_t)) g_t C_t), so that a state costs one exponential and three multiplications a token, a third of the walk's. Step
// sizes are summed anew for each tile, and the tiles' sums with their rounding kept: the exponents of slow states are
// differences of what would otherwise be long sums of equal terms.
template <typename T, int LPC, bool BACK>
__global__ void __launch_bounds__(kSelThreads, LPC <= 8 ? 3 : 2) sel_seg_kernel(const SelParams p) {
    using P = Place<T, LPC>;
    constexpr int kNp = 4 * LPC, V = P::kV, kCh = P::kCh;
    extern __shared__ __align__(16) unsigned char smem[];
    float2* sdt = reinterpret_cast<float2*>(smem);               // [tile][channels]: dt, dt u (BACK: g)
    float* sB = reinterpret_cast<float*>(sdt + kSelTile * kCh);  // [tile][states]: B (BACK: C)
    float* sbias = sB + kSelTile * kNp;
    T* raw = reinterpret_cast<T*>(sbias + kCh) + threadIdx.x * V;  // two turns of dt and u (BACK: dt, dout, z)
    constexpr int kRaw = kSelTile * kCh;
    const P at(p);
    const int seg = BACK ? blockIdx.y + 1 : blockIdx.y, first = seg * p.seg_tokens, last = min(p.L, first + p.seg_tokens);
    const int lane = threadIdx.x & 31, q = lane & (LPC - 1), ch = threadIdx.x / LPC, cp = pair_at(ch), d = at.d0 + ch;
    const bool in = ch < at.nch;
    constexpr int kBytes = need_vec<V * (int)sizeof(T)>();
    const SelTensor& x1 = BACK ? p.dout : p.u;
    const bool even = at.d0 % V == 0;
    const bool v1 = even && x1.vec >= kBytes, vd = even && p.dt.vec >= kBytes, vz = even && p.z.vec >= kBytes;
    States<T, LPC> Bs;
    auto load = [&](int l0, int turn) {
        const int l = l0 + at.row;
        if (l < last && at.left > 0) {
            T* to = raw + turn * 3 * kRaw;
            fetch<T, V>(to, row_of<T>(p.dt, at.b, l, at.d0 + at.c0), at.left, vd);
            fetch<T, V>(to + kRaw, row_of<T>(x1, at.b, l, at.d0 + at.c0), at.left, v1);
            if (BACK && p.z.p) fetch<T, V>(to + 2 * kRaw, row_of<T>(p.z, at.b, l, at.d0 + at.c0), at.left, vz);
        }
        fetch_commit();
        Bs.load(p, BACK ? p.C : p.Bm, at.b, at.g, l0, last);
    };
    const int tiles = (last - first + kSelTile - 1) / kSelTile;
    auto begin = [&](int i) { return first + (BACK ? i : tiles - 1 - i) * kSelTile; };
    load(begin(0), 0);
    for (int i = threadIdx.x; i < kCh; i += kSelThreads) sbias[i] = i < at.nch && p.dt_bias ? p.dt_bias[at.d0 + i] : 0.f;
    float A2[4];
    load_A<LPC>(p, d, in, q, A2);
    const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
    F2 h01 = f2(0.f), h23 = f2(0.f);
    float sum = 0.f, rest = 0.f;
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
        const int l0 = begin(i), l = l0 + at.row, turn = i & 1;
        const bool live = l < last && live_at<T>(p, at.b, l);
        const T* mine = raw + turn * 3 * kRaw;
        fetch_wait<0>();
        {
            Piece<T, V> dt, x, z;
            float s[V], g[V];
            dt.load(mine, V, true);
            x.load(mine + kRaw, V, true);
#pragma unroll
            for (int k = 0; k < V; ++k) s[k] = to_f<T>(dt.x[k]) + sbias[at.c0 + k];
            if (p.softplus) softplus_all(s);
            if (BACK && p.z.p) {
                z.load(mine + 2 * kRaw, V, true);
#pragma unroll
                for (int k = 0; k < V; ++k) g[k] = to_f<T>(z.x[k]);
                sigmoid_all(g);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float y = to_f<T>(x.x[k]);
                if (!BACK) y *= s[k];
                else if (p.z.p) y *= to_f<T>(z.x[k]) * g[k];
                const bool has = live && k < at.left;
                s[k] = has ? s[k] : 0.f;
                g[k] = has ? y : 0.f;
            }
            put_pairs(sdt + at.row * kCh, at.c0, s, g);
        }
        Bs.put(sB);
        if (i + 1 < tiles) load(begin(i + 1), turn ^ 1);
        __syncthreads();
        F2 t01 = f2(0.f), t23 = f2(0.f);
        float cum = 0.f;
#pragma unroll 8
        for (int k = 0; k < kSelTile; ++k) {
            const int t = BACK ? k : kSelTile - 1 - k;
            const float2 s = sdt[t * kCh + cp];
            const float4 Bv = *reinterpret_cast<const float4*>(sB + t * kNp + 4 * q);
            if (BACK) cum += s.x;
            const F2 y01 = mul(f2(cum), A01), y23 = mul(f2(cum), A23);
            float y[4];
            get(y01, y[0], y[1]);
            get(y23, y[2], y[3]);
            t01 = fma(f2(ex2(y[0]), ex2(y[1])), mul(f2(s.y), f2(Bv.x, Bv.y)), t01);
            t23 = fma(f2(ex2(y[2]), ex2(y[3])), mul(f2(s.y), f2(Bv.z, Bv.w)), t23);
            if (!BACK) cum += s.x;
        }
        // behind the tiles that have been summed (weighted as far as these reach)
        const float far = sum + rest;
        float s[4];
        get(t01, s[0], s[1]);
        get(t23, s[2], s[3]);
        if (fabsf(s[0]) + fabsf(s[1]) + fabsf(s[2]) + fabsf(s[3]) < INFINITY) {
            float y[4] = {A2[0] * far, A2[1] * far, A2[2] * far, A2[3] * far};
            if (fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) > 127.f) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = split_growth(y[j], s[j]);
                t01 = f2(s[0], s[1]);
                t23 = f2(s[2], s[3]);
            }
            h01 = fma(f2(ex2(y[0]), ex2(y[1])), t01, h01);
            h23 = fma(f2(ex2(y[2]), ex2(y[3])), t23, h23);
        } else {  // a state that grows past 2^127 within the tile: each token by itself, its whole factor in two steps
            float h[4];
            get(h01, h[0], h[1]);
            get(h23, h[2], h[3]);
            cum = 0.f;
#pragma unroll 1
            for (int k = 0; k < kSelTile; ++k) {
                const int t = BACK ? k : kSelTile - 1 - k;
                const float2 x = sdt[t * kCh + cp];
                const float4 Bv = *reinterpret_cast<const float4*>(sB + t * kNp + 4 * q);
                const float B4[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
                if (BACK) cum += x.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y = A2[j] * (cum + far);
                    const float v = split_growth(y, x.y * B4[j]);
                    h[j] = fmaf(ex2(y), v, h[j]);
                }
                if (!BACK) cum += x.x;
            }
            h01 = f2(h[0], h[1]);
            h23 = f2(h[2], h[3]);
        }
        add_exactly(sum, rest, cum);
        __syncthreads();
    }
    const int64_t to = ((int64_t)seg * p.B + at.b) * p.D + d;
    float h[4];
    get(h01, h[0], h[1]);
    get(h23, h[2], h[3]);
    if (in) {
        *reinterpret_cast<float4*>(p.seg_h + to * kNp + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
        if (q == 0) p.seg_dt[to] = sum + rest;
    }
}

// Token by token, without shared memory: a lane has four states of a channel and reads its token's values by itself. For
// single tokens (bound by the states' 8 N D bytes a sequence, or the launch) and calls of a few. WHOLE: four states are 16
// bytes of the state and of A, and a piece of B and C.
template <typename T, int LPC, bool WHOLE>
__global__ void __launch_bounds__(kSelThreads) sel_step_kernel(const SelParams p) {
    const int q = threadIdx.x & (LPC - 1), b = blockIdx.y;
    const int d = (int)(blockIdx.x * (kSelThreads / LPC) + threadIdx.x / LPC);
    const bool in = d < p.D, has = in && 4 * q < p.N;
    const int64_t g = p.G == 1 || !in ? 0 : d / p.Dg;
    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t sat = ((int64_t)b * p.D + d) * p.N + 4 * q;
    if (WHOLE) {
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
    const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
    F2 h01 = f2(h[0], h[1]), h23 = f2(h[2], h[3]);
    for (int l = 0; l < p.L; ++l) {
        const bool live = in && live_at<T>(p, b, l);
        float y = 0.f, u = 0.f, z = 0.f;
        if (live) {
            Piece<T, 4> Bp, Cp;
            Bp.zero();
            Cp.zero();
            const T* Bat = row_of<T>(p.Bm, b, l, 0) + g * p.Bm.sg + 4 * q;
            const T* Cat = row_of<T>(p.C, b, l, 0) + g * p.C.sg + 4 * q;
            if (has) {
                if (WHOLE) {
                    Bp.load(Bat);
                    Cp.load(Cat);
                } else {
                    Bp.load(Bat, p.N - 4 * q, false);
                    Cp.load(Cat, p.N - 4 * q, false);
                }
            }
            u = to_f<T>(*row_of<T>(p.u, b, l, d));
            float dt = to_f<T>(*row_of<T>(p.dt, b, l, d)) + bias;
            if (p.z.p) z = to_f<T>(*row_of<T>(p.z, b, l, d));
            if (p.softplus) dt = softplus(dt);
            const F2 dt2 = f2(dt), du = f2(dt * u);
            h01 = fma(du, f2(to_f<T>(Bp.x[0]), to_f<T>(Bp.x[1])), decayed(factor(mul(dt2, A01)), h01));
            h23 = fma(du, f2(to_f<T>(Bp.x[2]), to_f<T>(Bp.x[3])), decayed(factor(mul(dt2, A23)), h23));
            y = both(fma(h23, f2(to_f<T>(Cp.x[2]), to_f<T>(Cp.x[3])), mul(h01, f2(to_f<T>(Cp.x[0]), to_f<T>(Cp.x[1])))));
        }
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (in && q == 0 && p.out.p) {
            y = fmaf(Dw, u, y);
            if (p.z.p) y *= z * sigmoid(z);
            *const_cast<T*>(row_of<T>(p.out, b, l, d)) = from_f<T>(live ? y : 0.f);
        }
    }
    if (has && p.S_out) {
        get(h01, h[0], h[1]);
        get(h23, h[2], h[3]);
        if (WHOLE) {
            *reinterpret_cast<float4*>(p.S_out + sat) = make_float4(h[0], h[1], h[2], h[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) p.S_out[sat + i] = h[i];
        }
    }
}

template <typename T, int LPC>
constexpr size_t fwd_smem() {
    constexpr size_t kCh = kSelThreads / LPC;
    return kSelTile * kCh * (8 + 6 * sizeof(T)) + (size_t)kSelTile * 4 * LPC * 8 + kCh * 8;
}

template <typename T, int LPC>
constexpr size_t seg_smem() {
    constexpr size_t kCh = kSelThreads / LPC;
    return kSelTile * kCh * (8 + 6 * sizeof(T)) + (size_t)kSelTile * 4 * LPC * 4 + kCh * 4;
}

// (more than 48 KB of shared memory have to be asked for)
template <typename K>
cudaError_t launch_sel(K* kernel, size_t smem, const SelParams& p, int segments, cudaStream_t st) {
    if (smem > 48 * 1024) {
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
    }
    const int kCh = sel_channels(p.N);
    kernel<<<dim3((unsigned)(p.B * p.G * ((p.Dg + kCh - 1) / kCh)), (unsigned)segments), kSelThreads, smem, st>>>(p);
    return cudaGetLastError();
}
template <typename F>
cudaError_t by_lanes(int N, F f) {
    switch (sel_lanes(N)) {
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        default: return f(std::integral_constant<int, 32>{});
    }
}

template <typename T>
cudaError_t launch_fwd(const SelParams& p, SelPass pass, cudaStream_t st) {
    return by_lanes(p.N, [&](auto lpc) {
        constexpr int LPC = decltype(lpc)::value;
        if (pass != kSelWalk) return launch_sel(sel_seg_kernel<T, LPC, false>, seg_smem<T, LPC>(), p, p.nseg - 1, st);
        return p.out.p ? launch_sel(sel_fwd_kernel<T, LPC, true>, fwd_smem<T, LPC>(), p, p.nseg, st)
                       : launch_sel(sel_fwd_kernel<T, LPC, false>, fwd_smem<T, LPC>(), p, p.nseg, st);
    });
}

template <typename T>
cudaError_t launch_step(const SelParams& p, cudaStream_t st) {
    return by_lanes(p.N, [&](auto lpc) {
        constexpr int LPC = decltype(lpc)::value;
        const dim3 grid((unsigned)((p.D + kSelThreads / LPC - 1) / (kSelThreads / LPC)), (unsigned)p.B);
        const int need = 4 * (int)sizeof(T);
        auto group_fits = [&](const SelTensor& t) { return t.vec >= need && t.sg * (int64_t)sizeof(T) % need == 0; };
        const bool whole = p.N % 4 == 0 && group_fits(p.Bm) && group_fits(p.C) &&
                           ((reinterpret_cast<uintptr_t>(p.S_in) | reinterpret_cast<uintptr_t>(p.S_out) | reinterpret_cast<uintptr_t>(p.A)) & 15) == 0;
        if (whole) sel_step_kernel<T, LPC, true><<<grid, kSelThreads, 0, st>>>(p);
        else sel_step_kernel<T, LPC, false><<<grid, kSelThreads, 0, st>>>(p);
        return cudaGetLastError();
    });
}

}  // namespace sel
}  // namespace subq
