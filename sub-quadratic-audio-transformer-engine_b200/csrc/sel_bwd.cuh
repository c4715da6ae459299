// Selective scan, backward. With g_t = dout_t silu(z_t) and the adjoint of the state
//   G_t = C_t g_t + a_{t+1} G_{t+1},
//   dC_t = sum_d h_t g_t,   dB_t = sum_d G_t dt_t u_t,   du_t = dt_t (B_t . G_t) + D g_t,
//   d dt_t = u_t (B_t . G_t) + sum_n A G_t a_t h_{t-1},   dA = sum_t dt_t G_t a_t h_{t-1},
//   dz_t = dout_t y_t silu'(z_t),   dD = sum_t g_t u_t,   d raw_t = d dt_t sigmoid(raw_t + bias),   dbias = sum_t d raw_t.
//
// One CTA walks its channels' tiles of 32 tokens from the last to the first. The forward left the state before every
// eighth token; from it eight tokens' a h and factors are formed forwards in registers and used up backwards, so that each
// exponential is formed once. dB and dC are sums over channels: over a warp's by shuffles that halve the values at each
// step (lanes hold their states in an order by which nothing has to be selected), over the CTA's warps in shared memory, over CTAs by a second launch, all in a fixed order. Sums over tokens (dA, dD,
// dbias) are added per eight tokens or tile with their rounding kept (two float32 a sum). Segments as in the forward.
//
// Bound by latency: 415 us of the 4 x 2048 x 1536 training step (168 instructions for 32 states of a token, beside 75 us for the
// segments and 210 us for the forward). Two CTAs an SM are what registers and shared memory allow, 3.9 warps a scheduler that
// wait for shuffles and shared memory and for the instruction before (issue slots 0.58 used, FMA pipe 41 %, ALU 36 %).
#pragma once

#include "sel_fwd.cuh"

namespace subq {
namespace sel {

// The order in which a lane holds its four states, n ^ order: lanes of channels with the upper bits set hold them swapped, so
// that in the sums over channels every lane keeps its first registers and gives its last ones, with nothing to select.
template <int LPC>
__device__ __forceinline__ int state_order(int lane) {
    return (LPC <= 16 && (lane & 16) ? 2 : 0) | (LPC <= 8 && (lane & 8) ? 1 : 0);
}
__device__ __forceinline__ void reorder(float (&x)[4], int order) {
    const float a[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = order & 1 ? a[i ^ 1] : a[i], hi = order & 1 ? a[i ^ 3] : a[i ^ 2];
        x[i] = order & 2 ? hi : lo;
    }
}
// Sums of dB (b) and dC (c) over the 32 / LPC channels of a warp. out: LPC / 4 values of this lane (channel_value names them).
template <int LPC>
__device__ __forceinline__ void channel_sums(F2 b01, F2 b23, F2 c01, F2 c23, int lane, float (&out)[LPC / 4]) {
    float b[4], c[4];
    get(b01, b[0], b[1]);
    get(b23, b[2], b[3]);
    get(c01, c[0], c[1]);
    get(c23, c[2], c[3]);
    if constexpr (LPC <= 16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            b[i] += __shfl_xor_sync(0xffffffffu, b[i + 2], 16);
            c[i] += __shfl_xor_sync(0xffffffffu, c[i + 2], 16);
        }
    }
    if constexpr (LPC <= 8) {
        b[0] += __shfl_xor_sync(0xffffffffu, b[1], 8);
        c[0] += __shfl_xor_sync(0xffffffffu, c[1], 8);
    }
    if constexpr (LPC == 4) {
        const bool up = lane & 4;
        out[0] = (up ? c[0] : b[0]) + __shfl_xor_sync(0xffffffffu, up ? b[0] : c[0], 4);
    } else {
        constexpr int n = LPC / 8;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            out[i] = b[i];
            out[n + i] = c[i];
        }
    }
}
// What value k of lane ln is: state n of dB (false) or dC (true).
template <int LPC>
__device__ __forceinline__ bool channel_value(int ln, int k, int& n) {
    const int quad = 4 * (ln & (LPC - 1));
    if constexpr (LPC == 4) {
        n = quad + state_order<LPC>(ln);
        return ln & 4;
    } else {
        constexpr int per = LPC / 8;
        n = quad + ((k % per) ^ state_order<LPC>(ln));
        return k >= per;
    }
}

// The adjoint that enters segment `seg` from behind: what the segments after it make of dS_out.
template <int LPC>
__device__ __forceinline__ void chain_back(const SelParams& p, int seg, int b, int d, int q, const float (&A2)[4], float (&g)[4]) {
    constexpr int kNp = 4 * LPC;
    for (int s = p.nseg - 1; s > seg; --s) {
        const int64_t at = ((int64_t)s * p.B + b) * p.D + d;
        const float4 x = *reinterpret_cast<const float4*>(p.seg_h + at * kNp + 4 * q);
        const float dt = p.seg_dt[at];
        g[0] = decayed(A2[0] * dt, g[0]) + x.x;
        g[1] = decayed(A2[1] * dt, g[1]) + x.y;
        g[2] = decayed(A2[2] * dt, g[2]) + x.z;
        g[3] = decayed(A2[3] * dt, g[3]) + x.w;
    }
}

template <typename T, int LPC>
struct BwdSmem {
    static constexpr int kCh = kSelThreads / LPC, kNp = 4 * LPC, kWarps = kSelThreads / 32, kVals = LPC / 4;
    float2 sdt[kSelTile * kCh];    // dt, u; then du, d raw
    float sg[kSelTile * kCh];      // g; then dz
    float sgz[kSelTile * kCh];     // dout silu'(z)
    float slope[kSelTile * kCh];   // d dt / d raw
    static constexpr int kOrders = LPC <= 8 ? 4 : LPC == 16 ? 2 : 1;  // copies of B and C, one for each order of a lane's states
    float sB[kOrders][kSelTile * kNp], sC[kOrders][kSelTile * kNp];
    float sbias[kCh];
    float red[kWarps][kSelKeep][32 * kVals];
    float4 kept[kSelTile / kSelKeep][kSelThreads];           // a thread's own: the states before every eighth token
    alignas(16) T raw[4][kSelTile * kCh];  // a thread's own pieces of u, dt, z, dout of the next tile
};

// RANGES: this launch has one range of every segment's tokens (an instance of its own: 1 to 5 % of the walk).
template <typename T, int LPC, bool RANGES>
__global__ void __launch_bounds__(kSelThreads, LPC <= 8 ? 2 : 1) sel_bwd_kernel(const SelParams p) {
    using P = Place<T, LPC>;
    using S = BwdSmem<T, LPC>;
    constexpr int kNp = 4 * LPC, V = P::kV, kCh = P::kCh, kVals = S::kVals;
    extern __shared__ __align__(16) unsigned char smem[];
    S& s = *reinterpret_cast<S*>(smem);
    const P at(p);
    const int seg = blockIdx.y, seg_first = seg * p.seg_tokens, seg_last = min(p.L, seg_first + p.seg_tokens);
    const int first = RANGES ? seg_first + p.range0 : seg_first, last = RANGES ? min(seg_last, first + p.range_tokens) : seg_last;
    if (RANGES && first >= last) return;  // (a last segment that is shorter than the others)
    const int row0 = RANGES ? seg * p.range_tokens - first : 0, rows = RANGES ? p.rows : p.L;  // a token's row in part_bc: row0 + token
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane & (LPC - 1), ch = threadIdx.x / LPC, cp = pair_at(ch), cs = single_at(ch), d = at.d0 + ch;
    const bool in = ch < at.nch;
    constexpr int kBytes = need_vec<V * (int)sizeof(T)>();
    const bool even = at.d0 % V == 0;
    const bool vu = even && p.u.vec >= kBytes, vd = even && p.dt.vec >= kBytes, vz = even && p.z.vec >= kBytes, vg = even && p.dout.vec >= kBytes;
    const bool vdu = even && p.du.vec >= kBytes, vdd = even && p.ddt.vec >= kBytes, vdz = even && p.dz.vec >= kBytes;
    const int64_t keeps = (p.L + kSelKeep - 1) / kSelKeep;
    const int turn = threadIdx.x * V;
    auto fetch_rows = [&](int l0) {
        const int l = l0 + at.row;
        if (l < last && at.left > 0) {  // (a masked token's piece is fetched, but not used)
            fetch<T, V>(s.raw[0] + turn, row_of<T>(p.u, at.b, l, at.d0 + at.c0), at.left, vu);
            fetch<T, V>(s.raw[1] + turn, row_of<T>(p.dt, at.b, l, at.d0 + at.c0), at.left, vd);
            if (p.z.p) fetch<T, V>(s.raw[2] + turn, row_of<T>(p.z, at.b, l, at.d0 + at.c0), at.left, vz);
            fetch<T, V>(s.raw[3] + turn, row_of<T>(p.dout, at.b, l, at.d0 + at.c0), at.left, vg);
        }
    };
    auto fetch_kept = [&](int l) {  // l: a multiple of kSelKeep
        if (in && l < last)
            fetch<float, 4>(reinterpret_cast<float*>(&s.kept[l / kSelKeep % (kSelTile / kSelKeep)][threadIdx.x]),
                            p.kept + (((int64_t)at.b * keeps + l / kSelKeep) * p.D + d) * kNp + 4 * q, 4, true);
    };
    States<T, LPC> Bs, Cs;
    auto load_states = [&](int l0) {
        Bs.load(p, p.Bm, at.b, at.g, l0, last);
        Cs.load(p, p.C, at.b, at.g, l0, last);
    };
    const int top = first + (last - 1 - first) / kSelTile * kSelTile;
    fetch_rows(top);
    for (int t8 = 0; t8 < kSelTile; t8 += kSelKeep) fetch_kept(top + t8);
    fetch_commit();
    load_states(top);
    for (int i = threadIdx.x; i < kCh; i += kSelThreads) s.sbias[i] = i < at.nch && p.dt_bias ? p.dt_bias[at.d0 + i] : 0.f;
    float A2[4], g0[4] = {0.f, 0.f, 0.f, 0.f};
    load_A<LPC>(p, d, in, q, A2);
    auto carried = [&] { return p.carry + (((int64_t)seg * p.B + at.b) * p.D + d) * kNp + 4 * q; };
    if (RANGES && in && last < seg_last) {
        const float4 x = *reinterpret_cast<const float4*>(carried());
        g0[0] = x.x, g0[1] = x.y, g0[2] = x.z, g0[3] = x.w;
    } else if (in) {
        if (p.dS_out)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < p.N) g0[i] = p.dS_out[((int64_t)at.b * p.D + d) * p.N + 4 * q + i];
        chain_back<LPC>(p, seg, at.b, d, q, A2, g0);
    }
    const int order = state_order<LPC>(lane);
    reorder(A2, order);
    reorder(g0, order);
    const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
    const float* myB = s.sB[S::kOrders == 2 ? order / 2 : order] + 4 * q;
    const float* myC = s.sC[S::kOrders == 2 ? order / 2 : order] + 4 * q;
    F2 P01 = f2(g0[0], g0[1]), P23 = f2(g0[2], g0[3]);  // a_{t+1} G_{t+1}
    const float Dw = in && p.Dw ? p.Dw[d] : 0.f;
    // the lane's sums over its tokens (q, q + 4, ...), and its states' over all of them
    float dD = 0.f, dD_rest = 0.f, db = 0.f, db_rest = 0.f;
    float dA[4] = {0.f, 0.f, 0.f, 0.f}, dA_rest[4] = {0.f, 0.f, 0.f, 0.f};
    if (RANGES && in && last < seg_last) {  // the ranges behind this one
        const int64_t part = (int64_t)at.b * p.nseg + seg;
        const float4 x = *reinterpret_cast<const float4*>(p.part_a + (part * p.D + d) * kNp + 4 * q);
        dA[0] = x.x, dA[1] = x.y, dA[2] = x.z, dA[3] = x.w;
        reorder(dA, order);
        if (q == 0) {
            dD = p.part_d[part * 2 * p.D + d];
            db = p.part_d[(part * 2 + 1) * p.D + d];
        }
    }
    __syncthreads();
    for (int l0 = top; l0 >= first; l0 -= kSelTile) {
        const int l = l0 + at.row;
        const bool live = l < last && live_at<T>(p, at.b, l);
        fetch_wait<0>();
        {
            Piece<T, V> u, dt, z, go;
            u.load(s.raw[0] + turn, V, true);
            dt.load(s.raw[1] + turn, V, true);
            go.load(s.raw[3] + turn, V, true);
            float x[V], g[V], uf[V], sl[V], gz[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = to_f<T>(dt.x[i]) + s.sbias[at.c0 + i];
                g[i] = to_f<T>(go.x[i]);
                gz[i] = 0.f;
                sl[i] = 1.f;
            }
            if (p.softplus) softplus_slope_all(x, sl);
            if (p.z.p) {
                z.load(s.raw[2] + turn, V, true);
#pragma unroll
                for (int i = 0; i < V; ++i) gz[i] = to_f<T>(z.x[i]);
                sigmoid_all(gz);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float zf = to_f<T>(z.x[i]), gs = g[i] * gz[i];
                    gz[i] = gs * fmaf(zf, 1.f - gz[i], 1.f);
                    g[i] = gs * zf;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool has = live && i < at.left;
                x[i] = has ? x[i] : 0.f;
                uf[i] = has ? to_f<T>(u.x[i]) : 0.f;
                g[i] = has ? g[i] : 0.f;
                gz[i] = has ? gz[i] : 0.f;
                sl[i] = has ? sl[i] : 0.f;
            }
            put_pairs(s.sdt + at.row * kCh, at.c0, x, uf);
            put_singles(s.sg + at.row * kCh, at.c0, g);
            put_singles(s.sgz + at.row * kCh, at.c0, gz);
            put_singles(s.slope + at.row * kCh, at.c0, sl);
        }
#pragma unroll
        for (int o = 0; o < S::kOrders; ++o) {
            Bs.put(s.sB[o], S::kOrders == 2 ? 2 * o : o);
            Cs.put(s.sC[o], S::kOrders == 2 ? 2 * o : o);
        }
        const bool more = l0 > first;
        if (more) {
            fetch_rows(l0 - kSelTile);
            load_states(l0 - kSelTile);
        }
        __syncthreads();
#pragma unroll 1
        for (int t8 = kSelTile - kSelKeep; t8 >= 0; t8 -= kSelKeep) {
            if (l0 + t8 < last) {  // (else every token there is behind the end: nothing of the adjoint changes)
                Factor f01[kSelKeep], f23[kSelKeep];
                F2 ah01[kSelKeep], ah23[kSelKeep];  // a_t h_{t-1}
                F2 h01 = f2(0.f), h23 = f2(0.f);
                if (in) {
                    const float4 k = s.kept[t8 / kSelKeep][threadIdx.x];
                    float x[4] = {k.x, k.y, k.z, k.w};
                    reorder(x, order);
                    h01 = f2(x[0], x[1]);
                    h23 = f2(x[2], x[3]);
                }
                float ys[2] = {0.f, 0.f};  // y of tokens q and 4 + q
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = 4 * half + j, t = t8 + i;
                        const float2 x = s.sdt[t * kCh + cp];
                        const float4 Bv = *reinterpret_cast<const float4*>(myB + t * kNp);
                        const F2 dt2 = f2(x.x), du2 = f2(x.x * x.y);
                        f01[i] = factor(mul(dt2, A01));
                        f23[i] = factor(mul(dt2, A23));
                        ah01[i] = decayed(f01[i], h01);
                        ah23[i] = decayed(f23[i], h23);
                        h01 = fma(du2, f2(Bv.x, Bv.y), ah01[i]);
                        h23 = fma(du2, f2(Bv.z, Bv.w), ah23[i]);
                        if (p.z.p) {
                            const float4 Cv = *reinterpret_cast<const float4*>(myC + t * kNp);
                            y[j] = both(fma(h23, f2(Cv.z, Cv.w), mul(h01, f2(Cv.x, Cv.y))));
                        }
                    }
                    if (p.z.p) ys[half] = lane_sums4<LPC>(y, lane);
                }
                F2 a01 = f2(0.f), a23 = f2(0.f);
                float gu = 0.f, dr = 0.f;
#pragma unroll
                for (int half = 1; half >= 0; --half) {
                    float bg[4], ag[4];
#pragma unroll
                    for (int j = 3; j >= 0; --j) {
                        const int i = 4 * half + j, t = t8 + i;
                        const float2 x = s.sdt[t * kCh + cp];
                        const float4 Bv = *reinterpret_cast<const float4*>(myB + t * kNp), Cv = *reinterpret_cast<const float4*>(myC + t * kNp);
                        const F2 g2 = f2(s.sg[t * kCh + cs]), dt2 = f2(x.x), du2 = f2(x.x * x.y);
                        const F2 G01 = fma(f2(Cv.x, Cv.y), g2, P01), G23 = fma(f2(Cv.z, Cv.w), g2, P23);
                        bg[j] = both(fma(G23, f2(Bv.z, Bv.w), mul(G01, f2(Bv.x, Bv.y))));
                        const F2 n01 = mul(G01, ah01[i]), n23 = mul(G23, ah23[i]);
                        ag[j] = both(fma(n23, A23, mul(n01, A01)));
                        a01 = fma(dt2, n01, a01);
                        a23 = fma(dt2, n23, a23);
                        float v[kVals];
                        channel_sums<LPC>(mul(G01, du2), mul(G23, du2), mul(fma(du2, f2(Bv.x, Bv.y), ah01[i]), g2), mul(fma(du2, f2(Bv.z, Bv.w), ah23[i]), g2), lane, v);
#pragma unroll
                        for (int k = 0; k < kVals; ++k) s.red[warp][i][k * 32 + lane] = v[k];
                        P01 = decayed(f01[i], G01);
                        P23 = decayed(f23[i], G23);
                    }
                    const float b4 = lane_sums4<LPC>(bg, lane), a4 = lane_sums4<LPC>(ag, lane);
                    __syncwarp();  // every lane of the channel has read these tokens' dt, u and g
                    if (q < 4) {   // what is left of token q of the four
                        const int t = t8 + 4 * half + q;
                        const float2 x = s.sdt[t * kCh + cp];
                        const float g = s.sg[t * kCh + cs];
                        const float ddt = fmaf(x.y, b4, a4 * 0.6931471805599453f) * s.slope[t * kCh + cs];
                        s.sdt[t * kCh + cp] = make_float2(fmaf(x.x, b4, Dw * g), ddt);
                        s.sg[t * kCh + cs] = s.sgz[t * kCh + cs] * fmaf(Dw, x.y, ys[half]);
                        gu = fmaf(g, x.y, gu);
                        dr += ddt;
                    }
                }
                add_exactly(dD, dD_rest, gu);
                add_exactly(db, db_rest, dr);
                float x[4];
                get(a01, x[0], x[1]);
                get(a23, x[2], x[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) add_exactly(dA[i], dA_rest[i], x[i]);
                __syncthreads();
                for (int i = threadIdx.x; i < kSelKeep * 32 * kVals; i += kSelThreads) {
                    const int t = i / (32 * kVals), k = i / 32 % kVals, ln = i & 31, tok = l0 + t8 + t;
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < S::kWarps; ++w) sum += s.red[w][t][k * 32 + ln];
                    int n;
                    const bool c = channel_value<LPC>(ln, k, n);
                    if (tok < last) p.part_bc[((((int64_t)at.block(p) * p.B + at.b) * rows + row0 + tok) * p.G + at.g) * (2 * kNp) + (c ? kNp : 0) + n] = sum;
                }
                __syncthreads();
            }
            if (more) fetch_kept(l0 - kSelTile + t8);
        }
        fetch_commit();
        if (l < last && at.left > 0) {
            float a[V], b[V];
            Piece<T, V> du, dd, dz;
            get_pairs(s.sdt + at.row * kCh, at.c0, a, b);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                du.x[i] = from_f<T>(a[i]);
                dd.x[i] = from_f<T>(b[i]);
            }
            du.store(const_cast<T*>(row_of<T>(p.du, at.b, l, at.d0 + at.c0)), at.left, vdu);
            dd.store(const_cast<T*>(row_of<T>(p.ddt, at.b, l, at.d0 + at.c0)), at.left, vdd);
            if (p.z.p) {
                get_singles(s.sg + at.row * kCh, at.c0, a);
#pragma unroll
                for (int i = 0; i < V; ++i) dz.x[i] = from_f<T>(a[i]);
                dz.store(const_cast<T*>(row_of<T>(p.dz, at.b, l, at.d0 + at.c0)), at.left, vdz);
            }
        }
        __syncthreads();  // the next tile takes the place of this one
    }
    float g[4];
    get(P01, g[0], g[1]);
    get(P23, g[2], g[3]);
    reorder(g, order);
    if (RANGES && in && first > seg_first) {
        *reinterpret_cast<float4*>(carried()) = make_float4(g[0], g[1], g[2], g[3]);
    } else if (in && seg == 0 && p.dS_in) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * q + i < p.N) p.dS_in[((int64_t)at.b * p.D + d) * p.N + 4 * q + i] = g[i];
    }
    const int64_t part = (int64_t)at.b * p.nseg + seg;
#pragma unroll
    for (int i = 0; i < 4; ++i) dA[i] += dA_rest[i];
    reorder(dA, order);
    if (in) *reinterpret_cast<float4*>(p.part_a + (part * p.D + d) * kNp + 4 * q) = make_float4(dA[0], dA[1], dA[2], dA[3]);
    float sums[2] = {q < 4 ? dD + dD_rest : 0.f, q < 4 ? db + db_rest : 0.f};
#pragma unroll
    for (int o = 1; o < LPC; o <<= 1)
#pragma unroll
        for (int k = 0; k < 2; ++k) sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], o);
    if (in && q < 2) p.part_d[(part * 2 + q) * p.D + d] = sums[q];
}

// dB and dC: the parts of a group's channel blocks, added in order.
template <typename T>
__global__ void __launch_bounds__(256) sel_sum_bc_kernel(const SelParams p, int np, int blocks) {
    const int64_t n = (int64_t)p.B * p.rows * p.G * 2 * np;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int state = (int)(i % np);
        if (state >= p.N) continue;
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < blocks; ++k) s += p.part_bc[k * n + i];
        int64_t r = i / np;
        const int which = (int)(r & 1);
        r >>= 1;
        const int g = (int)(r % p.G);
        r /= p.G;
        int64_t l = r % p.rows;
        const int64_t b = r / p.rows;
        if (p.carry) {  // one range of several
            const int seg = (int)l / p.range_tokens;
            l += p.range0 + (int64_t)seg * (p.seg_tokens - p.range_tokens);
            if (l >= min((int64_t)p.L, (int64_t)(seg + 1) * p.seg_tokens)) continue;
        }
        if (which) static_cast<T*>(p.dC)[b * p.dC_sb + l * p.dC_sl + g * p.dC_sg + state] = from_f<T>(s);
        else static_cast<T*>(p.dB)[b * p.dB_sb + l * p.dB_sl + g * p.dB_sg + state] = from_f<T>(s);
    }
}

// dA, dD and dbias: the parts of sequences and segments, added in order.
template <typename T>
__global__ void __launch_bounds__(256) sel_sum_weights_kernel(const SelParams p, int np) {
    const int64_t n = (int64_t)p.D * (np + 2), parts = (int64_t)p.B * p.nseg;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t na = (int64_t)p.D * np;
        float s = 0.f, rest = 0.f;
        if (i < na) {
            if (i % np >= p.N) continue;
#pragma unroll 4
            for (int64_t k = 0; k < parts; ++k) add_exactly(s, rest, p.part_a[k * na + i]);
            p.dA[i / np * p.N + i % np] = s + rest;
        } else {
            const int64_t j = i - na;
            const int which = j >= p.D;
            float* to = which ? p.dbias : p.dD;
            if (!to) continue;
#pragma unroll 4
            for (int64_t k = 0; k < parts; ++k) add_exactly(s, rest, p.part_d[k * 2 * p.D + j]);
            to[j - (which ? p.D : 0)] = s + rest;
        }
    }
}

template <typename T>
cudaError_t launch_bwd(const SelParams& p, SelPass pass, cudaStream_t st) {
    return by_lanes(p.N, [&](auto lpc) {
        constexpr int LPC = decltype(lpc)::value;
        if (pass != kSelWalk) return launch_sel(sel_seg_kernel<T, LPC, true>, seg_smem<T, LPC>(), p, p.nseg - 1, st);
        return p.carry ? launch_sel(sel_bwd_kernel<T, LPC, true>, sizeof(BwdSmem<T, LPC>), p, p.nseg, st)
                       : launch_sel(sel_bwd_kernel<T, LPC, false>, sizeof(BwdSmem<T, LPC>), p, p.nseg, st);
    });
}

template <typename T>
cudaError_t launch_sums(const SelParams& p, bool weights, cudaStream_t st) {
    const int np = 4 * sel_lanes(p.N), kCh = sel_channels(p.N), blocks = (p.Dg + kCh - 1) / kCh;
    auto grid = [](int64_t n) { return (unsigned)((n + 255) / 256 < 148 * 16 ? (n + 255) / 256 : 148 * 16); };
    sel_sum_bc_kernel<T><<<grid((int64_t)p.B * p.rows * p.G * 2 * np), 256, 0, st>>>(p, np, blocks);
    if (weights) sel_sum_weights_kernel<T><<<grid((int64_t)p.D * (np + 2)), 256, 0, st>>>(p, np);
    return cudaGetLastError();
}

}  // namespace sel
}  // namespace subq
