// Backward of the gated delta rule from what the forward stored per chunk (Y,
// the state S0 before it, the corrections W). With G the gradient of the state
// after a chunk, D = e^{g_C - g}, dO the upstream gradient and P = scale G_ij q_i.k_j:
//   dU = P^T dO + D (K G),   Z = dU - Y^T (beta dU),
//   G0 = e^{g_C} G + scale (e^g Q)^T dO - K^T (e^g beta Z)
// is the walk back over the chunks (delta_rev_kernel, the mirror image of the
// forward's), and, with D1_ij = scale G_ij beta_j dO_i.W_j (i >= j) and
// D2_ij = -G_ij beta_i beta_j Z_i.W_j (i > j),
//   dQ = scale e^g (dO S0^T) + D1 K
//   dK = D beta (W G^T) - e^g beta (Z S0^T) + D1^T Q + D2^T K + D2 K
//   dV = beta Z,   dbeta_i = W_i.Z_i
// for all chunks at once (delta_grad_kernel). log gamma_t (token t of the chunk)
// scales every term that joins something before t to something from t on:
//   dlog gamma_t = sum over i >= t > j of E_ij + sum over i >= t of a_i + sum over j < t of b_j + e^{g_C} <G, S0>,
//   E_ij = D1_ij q_i.k_j + D2_ij k_i.k_j,   a_i = scale e^{g_i} q_i.(S0 dO_i) - e^{g_i} beta_i k_i.(S0 Z_i),
//   b_j = e^{g_C - g_j} beta_j k_j.(G W_j).
// From the end of the chunk backwards the first two are a running sum that row t of E
// and a_t enter and column t of E leaves, the very same numbers: what they are off by
// leaves with them, and what is left is the error of the terms that count for t. The
// third is a running sum from the begin of the chunk: all of b less those from t on
// would keep what b_j of late tokens, which may be large, are off by. (The shorter
// running sum of q_i.dq_i - v_i.dv_i is the same in exact arithmetic, but keeps the
// errors of tokens that have nothing to do with t: six times as far off with fast
// decay.)
//
// Measured, bf16, d = e = 64, 8 x 8 heads of 8192 tokens (8192 chunks): the walk back
// 396 us (3.1 us a chunk, bound like the forward's by shared memory, 60 % busy, and
// the latency of its three products in a row; few sequences are cut into segments, see
// delta_join.cuh and the rule in capi.cu), the gradients 543 us (140 KB read and
// written a chunk, 0.32 of measured HBM; tensor pipe 38 %, shared memory 53 %, 16
// warps per SM, whose 128 registers a thread spill 168 bytes).
#pragma once

#include "delta_common.cuh"
#include "delta_join.cuh"
#include "delta_launch.h"

namespace subq {
namespace {

using namespace dl;

// ------------------------------------------------------------------ the walk back
template <typename T, int DP>
struct RevSmem {
    static constexpr int kIn = kDeltaIn<T>, kX = kDeltaPlanes;
    // chunks in shared memory: the one at work and the next, where they fit one more on its way
    static constexpr int kStages = kIn == 1 ? (DP == 64 ? 3 : 2) : DP == 64 ? 2 : 1;
    struct Stage {
        alignas(128) unsigned char k[kIn * 64 * DP * 2];
        alignas(128) unsigned char q[kIn * 64 * DP * 2];
        alignas(128) unsigned char g[kIn * 64 * kDeltaCols * 2];  // dO
        alignas(128) unsigned char y[kX * kYBlocks * 512];
        alignas(128) unsigned char P[kX * kYBlocks * 512];  // scale G o (Q K^T)
        Gates s;
    } st[kStages];
    // by pair of warps
    alignas(16) unsigned char G[2][DP / 16][kX * 512];  // G^T, planes
    alignas(16) unsigned char R[2][4][kX * 512];        // -(beta dU)^T, planes
    // as W in the forward's walk: planes of -e^g beta Z and of Z, or Z in float32
    static constexpr bool kShared = kIn < 3;
    alignas(16) unsigned char Zk[2][kShared ? 4 : 1][kX * 512];
    union {
        float4 Z[2][kShared ? 1 : 8 * 32];
        unsigned char Zp[2][kShared ? 4 : 1][kX * 512];
    } z;
    float4 e2[2][DP / 8 * 32];                          // (scale (e^g Q)^T dO)^T; before that, (P^T dO)^T of the same chunk
};

// One warp of a chain pair: half `A` of d of G^T in its accumulators; dU and Z of its token blocks.
template <typename T, int DP, bool STATES>
__device__ __forceinline__ void rev_chain_warp(RevSmem<T, DP>& sm, const WalkJob& job, int A, int pair, int lane) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes, NST = RevSmem<T, DP>::kStages;
    constexpr int NH = DP / 16;
    constexpr bool kShared = RevSmem<T, DP>::kShared;
    const int g = lane >> 2, t = lane & 3;
    const Own own(A);
    const float2 one = make_float2(1.f, 1.f);
    float S[NH][4];  // G^T: 16 value columns x this half of d
    const int col0 = job.c0 + 16 * pair;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 8 * (A * NH + n) + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
            S[n][i] = job.ident ? (d == col ? 1.f : 0.f) : job.in && d < job.rows && col < job.ld ? job.in[(int64_t)d * job.ld + col] : 0.f;
        }
    auto put_state = [&]() {
#pragma unroll
        for (int kk = 0; kk < NH / 2; ++kk) {
            uint32_t a[NX][4];
            to_a<NX>(S[2 * kk], S[2 * kk + 1], one, one, a);
            put_a<NX>(sm.G[pair][A * (NH / 2) + kk], a, lane);
        }
    };
    put_state();
    __syncthreads();
    for (int c = job.end - 1; c >= job.begin; --c) {
        if (NST == 1) __syncthreads();
        auto& st = sm.st[c % NST];
        const Gates& s = st.s;
        if (s.any) {
            const uint32_t kt = smem_addr(st.k), yt = smem_addr(st.y) + lane * 16;
            float X[4][4];  // (K G)^T, then dU^T, then Z^T: blocks 2 u + half of this warp's tokens
            zero_acc<4>(X);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a[NX][4];
                get_a<NX>(a, sm.G[pair][kk], lane);
                mma_rows<DP, NX, NIN, NX>(X, a, kt, 16 * own.b0, 16 * own.b1, kk, lane);
            }
            bar_sync(1, 256);  // P^T dO is there; G has been read
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // dU; -beta dU for both warps
                const int tok = 16 * own.at(u) + 2 * t;
                float2 be[2];
#pragma unroll
                for (int jh = 0; jh < 2; ++jh) {
                    const float4 e1 = sm.e2[pair][(2 * own.at(u) + jh) * 32 + lane];
                    const float2 kd = *reinterpret_cast<const float2*>(&s.kd[tok + 8 * jh]);
                    be[jh] = *reinterpret_cast<const float2*>(&s.beta[tok + 8 * jh]);
                    be[jh] = make_float2(-be[jh].x, -be[jh].y);
                    float(&x)[4] = X[2 * u + jh];
                    x[0] = fmaf(kd.x, x[0], e1.x);
                    x[1] = fmaf(kd.y, x[1], e1.y);
                    x[2] = fmaf(kd.x, x[2], e1.z);
                    x[3] = fmaf(kd.y, x[3], e1.w);
                }
                uint32_t a[NX][4];
                to_a<NX>(X[2 * u], X[2 * u + 1], be[0], be[1], a);
                put_a<NX>(sm.R[pair][own.at(u)], a, lane);
            }
            bar_arrive(6 + pair, 128);  // P^T dO has been read: e2 may take its place
            bar_sync(4 + pair, 64);
#pragma unroll
            for (int ib = 0; ib < 4; ++ib) {  // Z^T = dU^T - (beta dU)^T Y
                if (ib < own.b0) continue;
                uint32_t a[NX][4];
                get_a<NX>(a, sm.R[pair][ib], lane);
                mma_blocks<NX, NX, false>(X, a, true, yt + tri(ib, own.b0) * 512, ib >= own.b1, yt + tri(ib, own.b1) * 512);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int jb = own.at(u);
                if constexpr (kShared) {
                    float2 f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 16 * jb + 8 * i + 2 * t;
                        const float2 be = *reinterpret_cast<const float2*>(&s.beta[j]), eg = *reinterpret_cast<const float2*>(&s.eg[j]);
                        f[i] = make_float2(-be.x * eg.x, -be.y * eg.y);
                    }
                    uint32_t a[NX][4];
                    to_a<NX>(X[2 * u], X[2 * u + 1], f[0], f[1], a);
                    put_a<NX>(sm.Zk[pair][jb], a, lane);
                    if constexpr (!STATES) {
                        to_a<NX>(X[2 * u], X[2 * u + 1], one, one, a);
                        put_a<NX>(sm.z.Zp[pair][jb], a, lane);
                    }
                } else {
                    sm.z.Z[pair][2 * jb * 32 + lane] = as_float4(X[2 * u]);
                    sm.z.Z[pair][(2 * jb + 1) * 32 + lane] = as_float4(X[2 * u + 1]);
                }
            }
            float U[NH][4];  // the chunk's part, summed by itself as in the forward's walk
            zero_acc<NH>(U);
            bar_sync(2, 256);  // Z is there for the pair and the warps beside it; e2 is there
#pragma unroll
            for (int n = 0; n < NH; ++n) add_acc(U[n], sm.e2[pair][(A * NH + n) * 32 + lane]);
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {  // G0^T = e^{g_C} G^T + e2 - (e^g beta Z)^T K over this half of d
                uint32_t a[NX][4];
                if constexpr (kShared) {
                    get_a<NX>(a, sm.Zk[pair][jb], lane);
                } else {
                    float z0[4], z1[4];
                    get_acc2(z0, z1, sm.z.Z[pair] + 2 * jb * 32, lane);
                    float2 f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 16 * jb + 8 * i + 2 * t;
                        const float2 be = *reinterpret_cast<const float2*>(&s.beta[j]), eg = *reinterpret_cast<const float2*>(&s.eg[j]);
                        f[i] = make_float2(-be.x * eg.x, -be.y * eg.y);
                    }
                    to_a<NX>(z0, z1, f[0], f[1], a);
                }
                mma_cols<NH, DP, NX, NIN, NX>(U, a, kt, 16 * jb, A * NH, lane);
            }
            next_state<NH>(S, s, U);
            put_state();
        }
        __syncthreads();
    }
    if (job.out) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 8 * (A * NH + n) + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
                if (d < job.rows && col < job.ld) job.out[job.ident ? (int64_t)col * job.ld + d : (int64_t)d * job.ld + col] = S[n][i];
            }
    }
}

// One warp of the pair beside a chain pair: P^T dO and dV for its token blocks, (e^g Q)^T dO for its half of d, and
// its share of the planes of G and Z.
template <typename T, int DP, bool STATES>
__device__ __forceinline__ void rev_side_warp(RevSmem<T, DP>& sm, const DeltaParams& p, const WalkJob& job, int A, int pair, int lane) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes, kGTile = 64 * kDeltaCols * 2;
    constexpr int NST = RevSmem<T, DP>::kStages, NH = DP / 16;
    const int g = lane >> 2, t = lane & 3, ncb = (p.e + kDeltaCols - 1) / kDeltaCols, cb = job.cb;
    const int64_t bh = job.bh;
    const Own own(A);
    const float2 one = make_float2(1.f, 1.f);
    constexpr int kPitch = 16 * sizeof(T) + 16, kPieces = 16 * sizeof(T) / 16;  // as the forward's staged outputs
    static_assert(4 * 32 * kPitch <= NX * kYBlocks * 512, "staged dv");
    const int col0 = cb * kDeltaCols + 16 * pair, width = min(16, p.e - col0);
    const bool whole = p.dv.vec && width == 16;
    T* dv = static_cast<T*>(p.dv.p) + tensor_base(p.dv, job.b, job.h);
    __syncthreads();
    for (int c = job.end - 1; c >= job.begin; --c) {
        if (NST == 1) __syncthreads();
        auto& st = sm.st[c % NST];
        const Gates& s = st.s;
        if (s.any) {
            const uint32_t qt = smem_addr(st.q), gt = smem_addr(st.g), pt = smem_addr(st.P) + lane * 16;
            const int64_t cw = (bh * p.nc + c) * 2 * ncb + 2 * cb + pair;  // chunk and group of 16 columns
            const int n0 = c * kDeltaC;
            float E[4][4];
            zero_acc<4>(E);
#pragma unroll
            for (int ib = 0; ib < 4; ++ib) {  // (P^T dO)^T
                if (ib < own.b0) continue;
                uint32_t a[NIN][4];  // dO^T: 16 value columns x 16 tokens
#pragma unroll
                for (int pl = 0; pl < NIN; ++pl) a_cols<kDeltaCols>(a[pl], gt + pl * kGTile, 16 * ib, pair, lane);
                mma_blocks<NIN, NX, true>(E, a, true, pt + tri(ib, own.b0) * 512, ib >= own.b1, pt + tri(ib, own.b1) * 512);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) sm.e2[pair][(2 * own.at(x >> 1) + (x & 1)) * 32 + lane] = as_float4(E[x]);
#pragma unroll
            for (int kk = 0; kk < (STATES ? 0 : DP / 16); ++kk) {
                if (kk % 2 != A) continue;
                uint32_t a[NX][4];
                get_a<NX>(a, sm.G[pair][kk], lane);
                store_matrices<NX>(p.dS + (cw * (DP / 16) + kk) * (NX * 512), a, lane);
            }
            bar_sync(1, 256);
            float E2[NH][4];
            zero_acc<NH>(E2);
#pragma unroll
            for (int ib = 0; ib < 4; ++ib) {
                uint32_t r[NIN][4], a[NX][4];
#pragma unroll
                for (int pl = 0; pl < NIN; ++pl) a_cols<kDeltaCols>(r[pl], gt + pl * kGTile, 16 * ib, pair, lane);
#pragma unroll
                for (int m = 0; m < 4; ++m) {  // scale e^g dO, tokens 16 ib + 8 (m / 2) + 2 t, + 1
                    float x = 0.f, y = 0.f;
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) {
                        const float2 u = unpack_bf16(r[pl][m]);
                        x += u.x;
                        y += u.y;
                    }
                    const float2 eg = *reinterpret_cast<const float2*>(&s.eg[16 * ib + 8 * (m >> 1) + 2 * t]);
                    uint32_t q[NX];
                    split2<NX>(x * (p.scale * eg.x), y * (p.scale * eg.y), q);
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl) a[pl][m] = q[pl];
                }
                mma_cols<NH, DP, NX, NIN, NX>(E2, a, qt, 16 * ib, A * NH, lane);
            }
            bar_sync(6 + pair, 128);
            put_acc<NH>(sm.e2[pair] + A * NH * 32, E2, lane);
            bar_sync(2, 256);
            // planes of Z, and dv = beta Z, staged where Y was (which nobody reads any more)
            unsigned char* stage = st.y + (2 * pair + A) * (32 * kPitch);
#pragma unroll
            for (int u = 0; u < (STATES ? 0 : 2); ++u) {
                uint32_t a[NX][4];
                float z0[4], z1[4];
                if constexpr (RevSmem<T, DP>::kShared) {
                    get_a<NX>(a, sm.z.Zp[pair][own.at(u)], lane);
                    from_a<NX>(z0, z1, a);
                } else {
                    get_acc2(z0, z1, sm.z.Z[pair] + 2 * own.at(u) * 32, lane);
                    to_a<NX>(z0, z1, one, one, a);
                }
                store_matrices<NX>(p.Z + (cw * 4 + own.at(u)) * (NX * 512), a, lane);
#pragma unroll
                for (int jh = 0; jh < 2; ++jh) {
                    const int tok = 16 * own.at(u) + 8 * jh + 2 * t;
                    const float2 be = *reinterpret_cast<const float2*>(&s.beta[tok]);
                    const float(&z)[4] = jh ? z1 : z0;
                    const float f[4] = {z[0] * be.x, z[1] * be.y, z[2] * be.x, z[3] * be.y};
                    if (p.dv32) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int n = n0 + tok + (i & 1), col = col0 + g + 8 * (i >> 1);
                            if (n < p.N && col < p.e) p.dv32[(bh * p.N + n) * p.e + col] = f[i];
                        }
                    } else {
                        T* r0 = reinterpret_cast<T*>(stage + (16 * u + 8 * jh + 2 * t) * kPitch);
                        T* r1 = reinterpret_cast<T*>(stage + (16 * u + 8 * jh + 2 * t + 1) * kPitch);
                        r0[g] = from_f<T>(f[0]);
                        r1[g] = from_f<T>(f[1]);
                        r0[g + 8] = from_f<T>(f[2]);
                        r1[g + 8] = from_f<T>(f[3]);
                    }
                }
            }
            if (!STATES && !p.dv32) {
                __syncwarp();
#pragma unroll
                for (int x = 0; x < kPieces; ++x) {
                    const int i = lane + 32 * x, row = i / kPieces, piece = i % kPieces;
                    const int tok = 16 * own.at(row >> 4) + (row & 15);
                    if (n0 + tok >= p.N) continue;
                    T* dst = dv + (n0 + tok) * p.dv.sn + col0;
                    const unsigned char* src = stage + row * kPitch + piece * 16;
                    if (whole) {
                        reinterpret_cast<uint4*>(dst)[piece] = *reinterpret_cast<const uint4*>(src);
                    } else {
                        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
                        for (int y = 0; y < kPer; ++y)
                            if (piece * kPer + y < width) dst[piece * kPer + y] = reinterpret_cast<const T*>(src)[y];
                    }
                }
            }
        }
        __syncthreads();
    }
}

// STATES: the gradients of the states alone, of segments that are walked side by side (delta_join.cuh). Segments count
// from the end; the last one's columns of the identity, as the first's results, nobody needs.
template <typename T, int DP, bool STATES>
__global__ void __launch_bounds__(384, 1) delta_rev_kernel(const DeltaParams p) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes;
    constexpr int NST = RevSmem<T, DP>::kStages;
    extern __shared__ __align__(128) unsigned char raw[];
    RevSmem<T, DP>& sm = *reinterpret_cast<RevSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols, ndb = STATES ? (p.d + kDeltaCols - 1) / kDeltaCols : 0, ncols = ncb + ndb;
    const int nseg = STATES ? p.nseg - 1 : p.nseg;
    const unsigned per_seq = (unsigned)(nseg * ncols - ndb), bh32 = blockIdx.x / per_seq;
    const int at = (int)(blockIdx.x - bh32 * per_seq) + ndb;  // (the last segment's columns at ndb ..)
    const int seg = at / ncols, col = at - seg * ncols;
    WalkJob job;
    job.bh = bh32;
    job.b = (int)(bh32 / (unsigned)p.H);
    job.h = (int)(bh32 - job.b * (unsigned)p.H);
    job.ident = STATES && col < ndb;
    job.cb = job.ident ? col : col - ndb;
    job.c0 = job.cb * kDeltaCols;
    job.begin = (p.nseg - 1 - seg) * p.seg_chunks;
    job.end = min(p.nc, job.begin + p.seg_chunks);
    job.ld = job.ident ? DP : p.e;
    job.rows = job.ident ? DP : p.d;
    const int64_t slot = job.bh * (p.nseg - 1) + seg;
    job.in = seg && !STATES ? p.seg_S + (slot - 1) * p.d * p.e : !seg && p.dS_out ? p.dS_out + job.bh * p.d * p.e : nullptr;
    if (STATES) job.out = job.ident ? p.seg_M + slot * (DP * DP) : p.seg_S + slot * p.d * p.e;
    else job.out = seg + 1 == nseg && p.dS_in ? p.dS_in + job.bh * p.d * p.e : nullptr;
    if (warp < 4) {
        rev_chain_warp<T, DP, STATES>(sm, job, warp & 1, warp >> 1, lane);
    } else if (warp < 8) {
        rev_side_warp<T, DP, STATES>(sm, p, job, warp & 1, (warp >> 1) & 1, lane);
    } else {  // ---------------------------------------------------------- loads
        const int lt = tid - 256;  // as in the forward's walk, from the last chunk to the first
        const int64_t bh = job.bh;
        const int b = job.b, h = job.h, begin = job.begin, end = job.end, c0 = job.c0;
        if (job.ident) {  // dO is 0 in every stage
            for (int i = 0; i < NST; ++i)
                for (int x = lt * 16; x < (int)sizeof(sm.st[i].g); x += 128 * 16)
                    *reinterpret_cast<uint4*>(sm.st[i].g + x) = make_uint4(0, 0, 0, 0);
        }
        const Gates* gates = p.gates + bh * p.nc;
        const int64_t kb = tensor_base(p.k, b, h), qb = tensor_base(p.q, b, h), gb = tensor_base(p.g, b, h);
        constexpr int kMat = NX * kYBlocks * 512;
        const unsigned char* Y = p.Y + bh * p.nc * kMat;
        const unsigned char* P = p.P + bh * p.nc * kMat;
        bool async = false;
        if constexpr (NIN == 1) async = p.k.vec && p.q.vec && p.g.vec && p.d % 8 == 0 && p.e % 8 == 0;
        if (async) {
            constexpr int kAhead = NST - 1;
            int any_next = gates[end - 1].any;
            auto start = [&](int c) {
                if (c >= begin) {
                    const int any = any_next;
                    any_next = c > begin ? gates[c - 1].any : 0;
                    auto& st = sm.st[c % NST];
                    async16<128>(reinterpret_cast<unsigned char*>(&st.s), reinterpret_cast<const unsigned char*>(gates + c), sizeof(Gates), lt);
                    if (any) {
                        const int n0 = c * kDeltaC;
                        async_tile<T, DP, 128>(st.k, p.k, kb, n0, 0, p.d, p.N, lt);
                        async_tile<T, DP, 128>(st.q, p.q, qb, n0, 0, p.d, p.N, lt);
                        if (!STATES || !job.ident) async_tile<T, kDeltaCols, 128>(st.g, p.g, gb, n0, c0, p.e, p.N, lt);
                        async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                        async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                    }
                }
                async_commit();
            };
            auto finish = [&](int c) {
                async_wait_but<(kAhead > 1 ? kAhead - 1 : 0)>();
                if (c < begin) return;
                bar_sync(3, 128);
                auto& st = sm.st[c % NST];
                if (st.s.any && !st.s.full) {
                    clear_dead<DP, 128>(st.k, st.s.live, lt);
                    clear_dead<DP, 128>(st.q, st.s.live, lt);
                    clear_dead<kDeltaCols, 128>(st.g, st.s.live, lt);
                }
            };
            for (int i = 1; i <= kAhead; ++i) start(end - i);
            finish(end - 1);
            __syncthreads();
            for (int c = end - 1; c >= begin; --c) {
                start(c - kAhead);
                finish(c - 1);
                __syncthreads();
            }
            async_wait();
        } else {
            if constexpr (NST == 1) {
                __syncthreads();
                for (int c = end - 1; c >= begin; --c) {
                    auto& st = sm.st[0];
                    copy16<128>(reinterpret_cast<unsigned char*>(&st.s), reinterpret_cast<const unsigned char*>(gates + c), sizeof(Gates), lt);
                    bar_sync(3, 128);
                    if (st.s.any) {
                        const int n0 = c * kDeltaC;
                        load_tile<T, DP, NIN, 128>(st.k, p.k, kb, n0, 0, p.d, p.N, st.s.live, lt);
                        load_tile<T, DP, NIN, 128>(st.q, p.q, qb, n0, 0, p.d, p.N, st.s.live, lt);
                        if (!STATES || !job.ident) load_tile<T, kDeltaCols, NIN, 128>(st.g, p.g, gb, n0, c0, p.e, p.N, st.s.live, lt);
                        async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                        async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                        async_wait();
                    }
                    __syncthreads();
                    __syncthreads();
                }
            } else {
                TileRegs<T, DP, 128> k, q;
                TileRegs<T, kDeltaCols, 128> x;
                ByteRegs<sizeof(Gates), 128> s;
                int any = 0, any_next = gates[end - 1].any;
                auto issue = [&](int c) {
                    any = any_next;
                    any_next = c > begin ? gates[c - 1].any : 0;
                    if (c < begin) return;
                    s.issue(gates + c, lt);
                    if (!any) return;
                    const int n0 = c * kDeltaC;
                    k.issue(p.k, kb, n0, 0, p.d, p.N, lt);
                    q.issue(p.q, qb, n0, 0, p.d, p.N, lt);
                    if (!STATES || !job.ident) x.issue(p.g, gb, n0, c0, p.e, p.N, lt);
                };
                auto store = [&](int c) {
                    if (c < begin) return;
                    auto& st = sm.st[c % NST];
                    s.store(&st.s, lt);
                    bar_sync(3, 128);
                    if (!any) return;
                    async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                    async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                    k.template store_planes<NIN>(st.k, st.s.live, lt);
                    q.template store_planes<NIN>(st.q, st.s.live, lt);
                    if (!STATES || !job.ident) x.template store_planes<NIN>(st.g, st.s.live, lt);
                };
                issue(end - 1);
                store(end - 1);
                issue(end - 2);
                async_wait();
                __syncthreads();
                for (int c = end - 1; c >= begin; --c) {
                    store(c - 1);
                    issue(c - 2);
                    async_wait();
                    __syncthreads();
                }
            }
        }
    }
}

// ------------------------------------------------------------------ the gradients
template <typename T, int DP>
struct GradSmem {
    static constexpr int kIn = kDeltaIn<T>, kX = kDeltaPlanes;
    static constexpr int kState = 2 * DP / 16 * kX * 512, kCol = 2 * 4 * kX * 512, kGTile = kIn * 64 * kDeltaCols * 2;
    // CTAs per SM (two with room for one block of 32 value columns each: 991 us for the backward of 8 x 8 heads of 8192
    // tokens in bf16; one with two blocks, or with more registers, 1140 and 1190)
    static constexpr int kCtas = sizeof(T) == 2 && DP == 64 ? 2 : 1;
    Gates s;
    float wz[kDeltaC];
    // halves (of d; D1's and D2's) of a_i, b_j and E's row sums, and E's column sums by block of rows
    float in[2][kDeltaC], out[2][kDeltaC], row[2][kDeltaC], col[2][4][kDeltaC];
    float gs[2];
    alignas(128) unsigned char k[kIn * 64 * DP * 2];
    alignas(128) unsigned char q[kIn * 64 * DP * 2];
    struct In {  // one block of 32 value columns
        alignas(128) unsigned char S0[kState];
        alignas(128) unsigned char G[kState];
        alignas(128) unsigned char W[kCol];
        alignas(128) unsigned char Z[kCol];
        alignas(128) unsigned char dO[kGTile];
    };
    struct Scores {
        alignas(128) unsigned char d1[kX * kYBlocks * 512];
        alignas(128) unsigned char d2[kX * kYBlocks * 512];
    };
    union {
        In in;
        Scores sc;
    } u;
};

// Rows of zeros.
template <typename T>
__device__ __forceinline__ void zero_rows(const DeltaTensor& x, int64_t base, float* x32, int64_t base32, int n0, int rows, int width, int tid) {
    for (int i = tid; i < rows * width; i += 256) {
        const int row = i / width, c = i % width;
        if (x32) x32[base32 + (int64_t)(n0 + row) * width + c] = 0.f;
        else (static_cast<T*>(x.p) + base + (n0 + row) * x.sn)[c] = from_f<T>(0.f);
    }
}

// Accumulators of 16 tokens (from n) x 8 NB columns (from c) to the rows of a gradient (`x32`, per state head, where given).
template <typename T, int NB>
__device__ __forceinline__ void store_grad(const float (&f)[NB][4], const DeltaTensor& x, int64_t base, float* x32, int64_t base32, int n,
                                           int end, int c, int width, int lane) {
    const int g = lane >> 2, t = lane & 3;
    c += 2 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = n + 8 * h + g;
        if (row >= end) continue;
        if (!x32 && x.vec && c - 2 * t + 8 * NB <= width) {  // rows start on 16 bytes and c is even
            T* at = static_cast<T*>(x.p) + base + row * x.sn + c;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                alignas(8) T v[2] = {from_f<T>(f[i][2 * h]), from_f<T>(f[i][2 * h + 1])};
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(at + 8 * i) = *reinterpret_cast<const uint32_t*>(v);
                else *reinterpret_cast<uint2*>(at + 8 * i) = *reinterpret_cast<const uint2*>(v);
            }
        } else {
            float* at32 = x32 ? x32 + base32 + (int64_t)row * width + c : nullptr;
            T* at = x32 ? nullptr : static_cast<T*>(x.p) + base + row * x.sn + c;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    if (c + 8 * i + y < width) {
                        if (x32) at32[8 * i + y] = f[i][2 * h + y];
                        else at[8 * i + y] = from_f<T>(f[i][2 * h + y]);
                    }
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(256, GradSmem<T, DP>::kCtas) delta_grad_kernel(const DeltaParams p) {
    using Smem = GradSmem<T, DP>;
    constexpr int NIN = Smem::kIn, NX = Smem::kX, kTile = 64 * DP * 2, kGTile = 64 * kDeltaCols * 2;
    constexpr int NB = DP / 16;  // 8-column blocks of a warp's half of d
    extern __shared__ __align__(128) unsigned char raw[];
    Smem& sm = *reinterpret_cast<Smem*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int rb = warp & 3, hf = warp >> 2;  // 16 tokens, half of d
    const unsigned chunk32 = blockIdx.x, bh32 = chunk32 / (unsigned)p.nc;  // (the grid fits 31 bits)
    const int64_t chunk = chunk32, bh = bh32;
    const int c = (int)(chunk32 - bh32 * p.nc), b = (int)(bh32 / (unsigned)p.H), h = (int)(bh32 - b * (unsigned)p.H), n0 = c * kDeltaC;
    const int rows = min(kDeltaC, p.N - n0);
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    const int64_t at32 = bh * p.N;  // rows of the gradients per state head
    const bool any = p.gates[chunk].any != 0;

    if (!any) {
        zero_rows<T>(p.dq, tensor_base(p.dq, b, h), p.dq32, at32 * p.d, n0, rows, p.d, tid);
        zero_rows<T>(p.dk, tensor_base(p.dk, b, h), p.dk32, at32 * p.d, n0, rows, p.d, tid);
        zero_rows<T>(p.dv, tensor_base(p.dv, b, h), p.dv32, at32 * p.e, n0, rows, p.e, tid);
        if (tid < rows) {
            p.dbeta[at32 + n0 + tid] = 0.f;
            if (p.dlg) p.dlg[at32 + n0 + tid] = 0.f;
        }
        return;
    }

    bool direct = false;  // bf16: tiles straight to shared memory
    if constexpr (NIN == 1) direct = p.k.vec && p.q.vec && p.g.vec && p.d % 8 == 0 && p.e % 8 == 0;
    auto start = [&](int eb) {  // the planes of a block of value columns
        auto& in = sm.u.in;
        const int64_t at = chunk * 2 * ncb + 2 * eb;
        async16<256>(in.S0, p.S0 + at * (Smem::kState / 2), Smem::kState, tid);
        async16<256>(in.G, p.dS + at * (Smem::kState / 2), Smem::kState, tid);
        async16<256>(in.W, p.W + at * (Smem::kCol / 2), Smem::kCol, tid);
        async16<256>(in.Z, p.Z + at * (Smem::kCol / 2), Smem::kCol, tid);
        if (direct) async_tile<T, kDeltaCols, 256>(in.dO, p.g, tensor_base(p.g, b, h), n0, eb * kDeltaCols, p.e, p.N, tid);
    };
    async16<256>(reinterpret_cast<unsigned char*>(&sm.s), reinterpret_cast<const unsigned char*>(p.gates + chunk), sizeof(Gates), tid);
    if (direct) {
        async_tile<T, DP, 256>(sm.k, p.k, tensor_base(p.k, b, h), n0, 0, p.d, p.N, tid);
        async_tile<T, DP, 256>(sm.q, p.q, tensor_base(p.q, b, h), n0, 0, p.d, p.N, tid);
    }
    start(0);
    const Gates& s = sm.s;
    async_wait();
    __syncthreads();
    if (!direct) {
        load_tile<T, DP, NIN, 256>(sm.k, p.k, tensor_base(p.k, b, h), n0, 0, p.d, p.N, s.live, tid);
        load_tile<T, DP, NIN, 256>(sm.q, p.q, tensor_base(p.q, b, h), n0, 0, p.d, p.N, s.live, tid);
    } else if (!s.full) {
        clear_dead<DP, 256>(sm.k, s.live, tid);
        clear_dead<DP, 256>(sm.q, s.live, tid);
    }

    float dq[NB][4], dk1[NB][4], dk2[NB][4], D[8][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) dq[n][i] = dk1[n][i] = dk2[n][i] = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) D[n][i] = 0.f;  // dO W^T (hf = 0) or Z W^T (hf = 1), rows 16 rb ..
    float ex[2][4];  // S0^T G of a group of 16 columns (hf = 1, rb < 2), of which the diagonal counts
    zero_acc<2>(ex);

    for (int eb = 0; eb < ncb; ++eb) {
        auto& in = sm.u.in;
        if (eb) {
            __syncthreads();  // the block before has been read
            start(eb);
        }
        if (!direct) load_tile<T, kDeltaCols, NIN, 256>(in.dO, p.g, tensor_base(p.g, b, h), n0, eb * kDeltaCols, p.e, p.N, s.live, tid);
        async_wait();
        if (direct && !s.full) {
            __syncthreads();
            clear_dead<kDeltaCols, 256>(in.dO, s.live, tid);
        }
        __syncthreads();
        const uint32_t S0 = smem_addr(in.S0) + lane * 16, G = smem_addr(in.G) + lane * 16;
        const uint32_t W = smem_addr(in.W) + lane * 16, Z = smem_addr(in.Z) + lane * 16;
        const uint32_t dO = smem_addr(in.dO);
#pragma unroll
        for (int cw = 0; cw < 2; ++cw) {  // 16 value columns: one k step
            uint32_t ao[NIN][4], a[NX][4];  // dO; Z, then W (one at a time: the accumulators leave no registers for both)
            auto load_a = [&](uint32_t from) {
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    uint32_t r[4];
                    ldm_t(r, from + ((cw * 4 + rb) * NX + pl) * 512);
                    a[pl][0] = r[0]; a[pl][1] = r[2]; a[pl][2] = r[1]; a[pl][3] = r[3];
                }
            };
            auto load_b = [&](uint32_t (&b0)[NX][2], uint32_t (&b1)[NX][2], uint32_t from) {
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    uint32_t r[4];
                    ldm_t(r, from + pl * 512);
                    b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                }
            };
#pragma unroll
            for (int pl = 0; pl < NIN; ++pl) a_rows<kDeltaCols>(ao[pl], dO + pl * kGTile, 16 * rb, cw, lane);
            load_a(Z);
#pragma unroll
            for (int n = 0; n < NB / 2; ++n) {
                uint32_t b0[NX][2], b1[NX][2];
                load_b(b0, b1, S0 + (cw * (DP / 16) + hf * (NB / 2) + n) * NX * 512);
                mma_pair<NIN, NX, NX>(dq[2 * n], dq[2 * n + 1], ao, b0, b1);
                mma_pair<NX, NX, NX>(dk2[2 * n], dk2[2 * n + 1], a, b0, b1);
            }
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {
                if (jb > rb) continue;
                uint32_t b0[NX][2], b1[NX][2];
                load_b(b0, b1, W + (cw * 4 + jb) * NX * 512);
                if (hf == 0) {
                    mma_pair<NIN, NX, NX>(D[2 * jb], D[2 * jb + 1], ao, b0, b1);
                } else {
                    mma_pair<NX, NX, NX>(D[2 * jb], D[2 * jb + 1], a, b0, b1);
                }
            }
            load_a(W);
#pragma unroll
            for (int n = 0; n < NB / 2; ++n) {
                uint32_t b0[NX][2], b1[NX][2];
                load_b(b0, b1, G + (cw * (DP / 16) + hf * (NB / 2) + n) * NX * 512);
                mma_pair<NX, NX, NX>(dk1[2 * n], dk1[2 * n + 1], a, b0, b1);
            }
            if (hf == 1 && rb == cw) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    uint32_t a[NX][4], b0[NX][2], b1[NX][2];
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl) {
                        uint32_t r[4];
                        ldm(a[pl], S0 + ((cw * (DP / 16) + kk) * NX + pl) * 512);
                        ldm(r, G + ((cw * (DP / 16) + kk) * NX + pl) * 512);
                        b0[pl][0] = r[0]; b0[pl][1] = r[2]; b1[pl][0] = r[1]; b1[pl][1] = r[3];
                    }
                    mma_pair<NX, NX, NX>(ex[0], ex[1], a, b0, b1);
                }
            }
        }
    }
    // diagonals: lanes with g = 2 t or 2 t + 1 have them
    const bool d0 = g == 2 * t, d1_ = g == 2 * t + 1;
    if (hf) {
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)  // W.Z
            if (jb == rb && (d0 || d1_)) {
                sm.wz[16 * rb + g] = d0 ? D[2 * jb][0] : D[2 * jb][1];
                sm.wz[16 * rb + 8 + g] = d0 ? D[2 * jb + 1][2] : D[2 * jb + 1][3];
            }
    }
    if (hf == 1 && rb < 2) {  // <G, S0>
        float gs = d0 ? ex[0][0] + ex[1][2] : d1_ ? ex[0][1] + ex[1][3] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) gs += __shfl_xor_sync(0xffffffffu, gs, o);
        if (lane == 0) sm.gs[rb] = gs;
    }
    __syncthreads();  // the blocks of value columns have been read: D1 and D2 take their place

    {  // D1 or D2 as planes; E's row and column sums
        unsigned char* dst = (hf ? sm.u.sc.d2 : sm.u.sc.d1) + lane * 4;
        const uint32_t at = smem_addr(hf ? sm.k : sm.q), kt = smem_addr(sm.k);
        float row[2] = {0.f, 0.f};
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
            if (jb > rb) continue;
            float sc[2][4];  // q_i.k_j or k_i.k_j
            zero_acc<2>(sc);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a[NIN][4], b0[NIN][2], b1[NIN][2];
#pragma unroll
                for (int pl = 0; pl < NIN; ++pl) {
                    uint32_t r[4];
                    a_rows<DP>(a[pl], at + pl * kTile, 16 * rb, kk, lane);
                    b_rows<DP>(r, kt + pl * kTile, 16 * jb, kk, lane);
                    b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                }
                mma_pair<NIN, NIN, NX>(sc[0], sc[1], a, b0, b1);
            }
#pragma unroll
            for (int jh = 0; jh < 2; ++jh) {
                const int j = 16 * jb + 8 * jh + 2 * t;
                const float2 be = *reinterpret_cast<const float2*>(&s.beta[j]);
                float2 col = make_float2(0.f, 0.f);
#pragma unroll
                for (int ih = 0; ih < 2; ++ih) {
                    const int i = 16 * rb + 8 * ih + g, keep = hf ? i - 1 : i;
                    const float fi = hf ? -s.beta[i] : p.scale;
                    const float2 ga = gamma_pair(s.gh[i], s.gl[i], s, j, keep);
                    const float x = fi * be.x * ga.x * select0(j <= keep, D[2 * jb + jh][2 * ih]);
                    const float y = fi * be.y * ga.y * select0(j + 1 <= keep, D[2 * jb + jh][2 * ih + 1]);
                    uint32_t r[NX];
                    split2<NX>(x, y, r);
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl)
                        *reinterpret_cast<uint32_t*>(dst + (pl * kYBlocks + tri(rb, jb)) * 512 + (ih * 2 + jh) * 128) = r[pl];
                    const float ex0 = select0(j < i, x * sc[jh][2 * ih]), ey0 = select0(j + 1 < i, y * sc[jh][2 * ih + 1]);
                    row[ih] += ex0 + ey0;
                    col.x += ex0;
                    col.y += ey0;
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    col.x += __shfl_xor_sync(0xffffffffu, col.x, o);
                    col.y += __shfl_xor_sync(0xffffffffu, col.y, o);
                }
                if (g == 0) *reinterpret_cast<float2*>(&sm.col[hf][rb][j]) = col;
            }
        }
#pragma unroll
        for (int ih = 0; ih < 2; ++ih) {
            row[ih] += __shfl_xor_sync(0xffffffffu, row[ih], 1);
            row[ih] += __shfl_xor_sync(0xffffffffu, row[ih], 2);
            if (t == 0) sm.row[hf][16 * rb + 8 * ih + g] = row[ih];
        }
    }
    // row factors of the products with the states; a_i and b_j
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int i = 16 * rb + 8 * x + g;
        const float fq = p.scale * s.eg[i], f1 = s.kd[i] * s.beta[i], f2 = -s.eg[i] * s.beta[i];
        float in = 0.f, out = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const uint32_t off = tile_off<DP>(i, hf * NB + n) + 4 * t;
            float2 kv = make_float2(0.f, 0.f), qv = kv;
#pragma unroll
            for (int pl = 0; pl < NIN; ++pl) {
                const float2 u = unpack_bf16(*reinterpret_cast<const uint32_t*>(sm.k + pl * kTile + off));
                const float2 w = unpack_bf16(*reinterpret_cast<const uint32_t*>(sm.q + pl * kTile + off));
                kv.x += u.x; kv.y += u.y;
                qv.x += w.x; qv.y += w.y;
            }
            const float2 d1 = make_float2(f1 * dk1[n][2 * x], f1 * dk1[n][2 * x + 1]);
            const float2 d2 = make_float2(f2 * dk2[n][2 * x], f2 * dk2[n][2 * x + 1]);
            dq[n][2 * x] *= fq;
            dq[n][2 * x + 1] *= fq;
            out = fmaf(d1.x, kv.x, fmaf(d1.y, kv.y, out));
            in = fmaf(d2.x, kv.x, fmaf(d2.y, kv.y, in));
            in = fmaf(dq[n][2 * x], qv.x, fmaf(dq[n][2 * x + 1], qv.y, in));
            dk1[n][2 * x] = d1.x + d2.x;
            dk1[n][2 * x + 1] = d1.y + d2.y;
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            in += __shfl_xor_sync(0xffffffffu, in, o);
            out += __shfl_xor_sync(0xffffffffu, out, o);
        }
        if (t == 0) {
            sm.in[hf][i] = in;
            sm.out[hf][i] = out;
        }
    }
    __syncthreads();
    const uint32_t d1 = smem_addr(sm.u.sc.d1) + lane * 16, d2 = smem_addr(sm.u.sc.d2) + lane * 16;
    const uint32_t kt = smem_addr(sm.k), qt = smem_addr(sm.q);
    constexpr int kP = kYBlocks * 512;
#pragma unroll
    for (int ob = 0; ob < 4; ++ob) {
        // D1 K and D2 K: tokens ob <= rb; D1^T Q and D2^T K: tokens ob >= rb
        uint32_t a1[NX][4], a2[NX][4], a1t[NX][4], a2t[NX][4];
#pragma unroll
        for (int pl = 0; pl < NX; ++pl) {
            uint32_t r[4];
            if (ob <= rb) {
                ldm(r, d1 + pl * kP + tri(rb, ob) * 512);
                a1[pl][0] = r[0]; a1[pl][1] = r[2]; a1[pl][2] = r[1]; a1[pl][3] = r[3];
                ldm(r, d2 + pl * kP + tri(rb, ob) * 512);
                a2[pl][0] = r[0]; a2[pl][1] = r[2]; a2[pl][2] = r[1]; a2[pl][3] = r[3];
            }
            if (ob >= rb) {
                ldm_t(a1t[pl], d1 + pl * kP + tri(ob, rb) * 512);
                ldm_t(a2t[pl], d2 + pl * kP + tri(ob, rb) * 512);
            }
        }
#pragma unroll
        for (int n = 0; n < NB / 2; ++n) {
            const int np = hf * (NB / 2) + n;
            uint32_t k0[NIN][2], k1[NIN][2], q0[NIN][2], q1[NIN][2];
#pragma unroll
            for (int pl = 0; pl < NIN; ++pl) {
                uint32_t r[4];
                b_cols<DP>(r, kt + pl * kTile, 16 * ob, np, lane);
                k0[pl][0] = r[0]; k0[pl][1] = r[1]; k1[pl][0] = r[2]; k1[pl][1] = r[3];
                b_cols<DP>(r, qt + pl * kTile, 16 * ob, np, lane);
                q0[pl][0] = r[0]; q0[pl][1] = r[1]; q1[pl][0] = r[2]; q1[pl][1] = r[3];
            }
            if (ob <= rb) {
                mma_pair<NX, NIN, NX>(dq[2 * n], dq[2 * n + 1], a1, k0, k1);
                mma_pair<NX, NIN, NX>(dk1[2 * n], dk1[2 * n + 1], a2, k0, k1);
            }
            if (ob >= rb) {
                mma_pair<NX, NIN, NX>(dk1[2 * n], dk1[2 * n + 1], a1t, q0, q1);
                mma_pair<NX, NIN, NX>(dk1[2 * n], dk1[2 * n + 1], a2t, k0, k1);
            }
        }
    }
    store_grad<T, NB>(dq, p.dq, tensor_base(p.dq, b, h), p.dq32, at32 * p.d, n0 + 16 * rb, n0 + rows, 8 * hf * NB, p.d, lane);
    store_grad<T, NB>(dk1, p.dk, tensor_base(p.dk, b, h), p.dk32, at32 * p.d, n0 + 16 * rb, n0 + rows, 8 * hf * NB, p.d, lane);
    __syncthreads();
    if (warp == 0) {
        // two tokens per lane: a_i and E from the end of the chunk backwards, b_j from its begin
        const int i0 = 2 * lane, i1 = i0 + 1, first = lane >> 3;
        float x[2], out[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = i0 + i;
            float col = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k >= first) col += sm.col[0][k][n] + sm.col[1][k][n];
            out[i] = sm.out[0][n] + sm.out[1][n];
            x[i] = (sm.in[0][n] + sm.in[1][n]) + (sm.row[0][n] + sm.row[1][n]) - col;
        }
        float run = x[0] + x[1], past = out[0] + out[1];  // over this lane's tokens and the later (earlier) lanes'
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float down = __shfl_down_sync(0xffffffffu, run, o), up = __shfl_up_sync(0xffffffffu, past, o);
            if (lane + o < 32) run += down;
            if (lane >= o) past += up;
        }
        float later = __shfl_down_sync(0xffffffffu, run, 1), before = __shfl_up_sync(0xffffffffu, past, 1);
        if (lane == 31) later = 0.f;
        if (lane == 0) before = 0.f;
        const float all = s.eC * (sm.gs[0] + sm.gs[1]);
        const float g1 = (x[1] + later) + (before + out[0]) + all, g0 = (x[0] + (x[1] + later)) + before + all;
        const int64_t at = at32 + n0;
        if (i0 < rows) {
            p.dbeta[at + i0] = s.live[i0] ? sm.wz[i0] : 0.f;
            if (p.dlg) p.dlg[at + i0] = s.live[i0] ? g0 : 0.f;
        }
        if (i1 < rows) {
            p.dbeta[at + i1] = s.live[i1] ? sm.wz[i1] : 0.f;
            if (p.dlg) p.dlg[at + i1] = s.live[i1] ? g1 : 0.f;
        }
    }
}

// x[b, hx, n, :] = sum over the group's state heads of x32, in head order
template <typename T>
__global__ void __launch_bounds__(256) delta_group_sum_kernel(const float* x32, DeltaTensor x, int H, int N, int width, int64_t total) {
    const int64_t at = blockIdx.x * (int64_t)256 + threadIdx.x;  // over [B, Hx, N, width]
    if (at >= total) return;
    const int col = (int)(at % width), hx = (int)(at / width / N % (H / x.group)), b = (int)(at / width / N / (H / x.group));
    const int64_t n = at / width % N;
    float s = 0.f;
    for (int i = 0; i < x.group; ++i) s += x32[((int64_t)(b * (int64_t)H + hx * x.group + i) * N + n) * width + col];
    static_cast<T*>(x.p)[b * x.sb + hx * x.sh + n * x.sn + col] = from_f<T>(s);
}

template <typename T>
cudaError_t group_sum(const float* x32, const DeltaTensor& x, const DeltaParams& p, int width, cudaStream_t st, int* launches) {
    if (!x32) return cudaSuccess;
    const int64_t total = (int64_t)p.B * (p.H / x.group) * p.N * width;
    delta_group_sum_kernel<T><<<(unsigned)((total + 255) / 256), 256, 0, st>>>(x32, x, p.H, p.N, width, total);
    ++*launches;
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t bwd_t(const DeltaParams& p, cudaStream_t st, int* launches) {
    const int64_t bh = (int64_t)p.B * p.H, ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    static_assert(sizeof(RevSmem<T, DP>) <= 227 * 1024 && sizeof(GradSmem<T, DP>) <= 227 * 1024, "shared memory");
    const size_t rev = sizeof(RevSmem<T, DP>), grad = sizeof(GradSmem<T, DP>);
    auto walk = [&](auto kernel, int64_t blocks) {
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rev);
        if (err != cudaSuccess) return err;
        kernel<<<(unsigned)blocks, 384, rev, st>>>(p);
        return cudaGetLastError();
    };
    cudaError_t err = cudaFuncSetAttribute(delta_grad_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)grad);
    if (err != cudaSuccess) return err;
    *launches = 2;
    if (p.nseg > 1) {
        const int64_t ndb = (p.d + kDeltaCols - 1) / kDeltaCols;
        if ((err = walk(delta_rev_kernel<T, DP, true>, bh * ((p.nseg - 1) * (ncb + ndb) - ndb))) != cudaSuccess) return err;
        if ((err = join_t<DP>(p, st)) != cudaSuccess) return err;
        *launches = 4;
    }
    if ((err = walk(delta_rev_kernel<T, DP, false>, bh * p.nseg * ncb)) != cudaSuccess) return err;
    delta_grad_kernel<T, DP><<<(unsigned)(bh * p.nc), 256, grad, st>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    if ((err = group_sum<T>(p.dq32, p.dq, p, p.d, st, launches)) != cudaSuccess) return err;
    if ((err = group_sum<T>(p.dk32, p.dk, p, p.d, st, launches)) != cudaSuccess) return err;
    return group_sum<T>(p.dv32, p.dv, p, p.e, st, launches);
}

}  // namespace
}  // namespace subq
