// Chunked forward of the gated delta rule (see delta_common.cuh for the algebra).
//
// delta_prep_kernel: gates, Y and scores of every chunk, all chunks at once.
// delta_chain_kernel: the walk over the chunks, bound by the latency of its
// dependent products (K S0, Y (beta R), K^T W per chunk). All products are
// transposed (rows = value columns, columns = tokens or d), so that a result is,
// in its registers, the A operand of the next product. A pair of warps owns 16
// value columns of one sequence: each warp forms R and W of two of the chunk's
// four blocks of 16 tokens and updates half of d of the state, float32 in its
// accumulators; the operands pass between the two through shared memory. Per
// CTA, 32 columns: two such pairs; two pairs of output warps (Q S0 and score W
// products; they also write the planes that the backward reads); and four warps
// that load the next chunks. Each SM sub-partition has one warp of each kind.
// (Four warps per 16 columns move each operand through shared memory twice as often
// and were slower.)
//
// Measured, bf16, d = e = 64, 8 x 8 heads of 8192 tokens (8192 chunks): gates and Y
// 128 us (issue-bound: 54 % of the issue slots with 20 warps per SM, tensor pipe 22 %);
// the walk 2.4 us a chunk, 2.7 us where the backward's planes are written (351 us:
// shared memory 70 % busy on the SMs at work, tensor pipe 43 %).
#pragma once

#include "delta_common.cuh"
#include "delta_join.cuh"
#include "delta_launch.h"
#include "scan_launch.h"

namespace subq {
namespace {

using namespace dl;

// ------------------------------------------------------------------ gates, Y and scores per chunk
template <typename T, int DP>
struct PrepSmem {
    static constexpr int kIn = kDeltaIn<T>, kX = kDeltaPlanes;
    Gates s;
    alignas(16) float A[kYBlocks][16][20];        // its lower triangle's blocks
    alignas(128) unsigned char Ab[6 * kX * 512];  // -A_IK beta, blocks I > K: [block][plane]
    alignas(128) unsigned char k[kIn * 64 * DP * 2];
    alignas(128) unsigned char q[kIn * 64 * DP * 2];
    // where (I + A_II beta)^-1 goes: over the 16 rows of q that warp I alone reads, once it has. (Five CTAs per SM then
    // have room for bf16 at d = 64.)
    static __host__ __device__ constexpr int ti(int I) { return (3 - I) * 16 * DP * 2; }
    static_assert(kX * 512 <= 16 * DP * 2, "T in q's rows");
};

// Y by 16 x 16 blocks. With T_I = (I + A_II beta)^-1 (forward substitution, a
// column per lane), block column J of Y is one warp's:
//   Y_JJ^T = A_JJ^T T_J^T,   Y_IJ^T = (A_IJ^T - sum_{J <= K < I} Y_KJ^T (A_IK beta)^T) T_I^T,
// transposed so that each result is, in its registers, the A operand of the next product.
template <typename T, int DP>
__global__ void __launch_bounds__(128) delta_prep_kernel(const DeltaParams p) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes, kTile = 64 * DP * 2;
    extern __shared__ __align__(128) unsigned char raw[];
    PrepSmem<T, DP>& sm = *reinterpret_cast<PrepSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const unsigned chunk32 = blockIdx.x, bh32 = chunk32 / (unsigned)p.nc;  // bh * nc + c (the grid fits 31 bits)
    const int64_t chunk = chunk32;
    const int c = (int)(chunk32 - bh32 * p.nc), b = (int)(bh32 / (unsigned)p.H), h = (int)(bh32 - b * (unsigned)p.H), n0 = c * kDeltaC;
    {
        TileRegs<T, DP, 128> k, q;
        k.issue(p.k, tensor_base(p.k, b, h), n0, 0, p.d, p.N, tid);
        q.issue(p.q, tensor_base(p.q, b, h), n0, 0, p.d, p.N, tid);
        if (warp == 0) form_gates(sm.s, p, b, h, n0, lane);
        __syncthreads();
        copy16<128>(reinterpret_cast<unsigned char*>(p.gates + chunk), reinterpret_cast<const unsigned char*>(&sm.s), sizeof(Gates), tid);
        if (!sm.s.any) return;  // nothing else of a dead chunk is read
        k.template store_planes<NIN>(sm.k, sm.s.live, tid);
        q.template store_planes<NIN>(sm.q, sm.s.live, tid);
    }
    __syncthreads();
    {  // A, rows 16 warp .. 16 warp + 15
        float acc[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
        const uint32_t k = smem_addr(sm.k);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            uint32_t a[NIN][4];
#pragma unroll
            for (int pl = 0; pl < NIN; ++pl) a_rows<DP>(a[pl], k + pl * kTile, 16 * warp, kk, lane);
#pragma unroll
            for (int jb = 0; jb < 4; ++jb)
                if (jb <= warp) {
                    uint32_t b0[NIN][2], b1[NIN][2];
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) {
                        uint32_t r[4];
                        b_rows<DP>(r, k + pl * kTile, 16 * jb, kk, lane);
                        b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                    }
                    mma_pair<NIN, NIN, NX>(acc[2 * jb], acc[2 * jb + 1], a, b0, b1);
                }
        }
#pragma unroll
        for (int ih = 0; ih < 2; ++ih) {
            const int i = 16 * warp + 8 * ih + g;
            const float gh = sm.s.gh[i], gl = sm.s.gl[i];
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (n <= 2 * warp + 1) {
                    const int j = 8 * n + 2 * t;
                    const float2 ga = gamma_pair(gh, gl, sm.s, j, i - 1);
                    const float x = ga.x * select0(j < i, acc[n][2 * ih]), y = ga.y * select0(j + 1 < i, acc[n][2 * ih + 1]);
                    *reinterpret_cast<float2*>(&sm.A[tri(warp, n >> 1)][8 * ih + g][j & 15]) = make_float2(x, y);
                    if (n < 2 * warp) {
                        const float2 be = *reinterpret_cast<const float2*>(&sm.s.beta[j]);
                        uint32_t r[NX];
                        split2<NX>(-be.x * x, -be.y * y, r);
                        unsigned char* at = sm.Ab + tri(warp - 1, n >> 1) * (NX * 512) + (ih * 2 + (n & 1)) * 128 + lane * 4;
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) *reinterpret_cast<uint32_t*>(at + pl * 512) = r[pl];
                    }
                }
        }
    }
    // scores, the longest rows where A's were the shortest
    score_rows<DP, NIN, NX>(p.P + chunk * (NX * kYBlocks * 512), smem_addr(sm.q), smem_addr(sm.k), sm.s, p.scale, 3 - warp, lane);
    __syncwarp();  // the diagonal block is this warp's own, as are the rows of q
    {
        const int col = lane & 15, r0 = 16 * warp;
        float ti[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // T e_col: t_i = delta - sum_j A_ij beta_j t_j, kept as beta_j t_j
            float x = i == col ? 1.f : 0.f, y = 0.f;
#pragma unroll
            for (int j = 0; j < i; j += 2) {
                const float2 a = *reinterpret_cast<const float2*>(&sm.A[tri(warp, warp)][i][j]);
                x = fmaf(-a.x, ti[j], x);
                if (j + 1 < i) y = fmaf(-a.y, ti[j + 1], y);
            }
            x += y;
            if (lane < 16) {
                unsigned char* at = sm.q + sm.ti(warp) + ((i >> 3) * 2 + (col >> 3)) * 128 + (i & 7) * 16 + (col & 7) * 2;
                float rest = x;
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    const __nv_bfloat16 u = __float2bfloat16_rn(rest);
                    *reinterpret_cast<__nv_bfloat16*>(at + pl * 512) = u;
                    rest -= __bfloat162float(u);
                }
            }
            ti[i] = sm.s.beta[r0 + i] * x;
        }
    }
    __syncthreads();
    {
        const int J = warp;
        uint32_t y[4][NX][4];  // Y_KJ^T, K = J + index
        unsigned char* Y = p.Y + chunk * (NX * kYBlocks * 512);
        const uint32_t ab = smem_addr(sm.Ab) + lane * 16, ti = smem_addr(sm.q) + lane * 16;
        const float2 one = make_float2(1.f, 1.f);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int I = J + x;
            if (I > 3) break;
            float acc[2][4], out[2][4];
#pragma unroll
            for (int ih = 0; ih < 2; ++ih)
#pragma unroll
                for (int v = 0; v < 4; ++v) {  // A_IJ^T: rows j, columns i
                    acc[ih][v] = sm.A[tri(I, J)][8 * ih + 2 * t + (v & 1)][g + 8 * (v >> 1)];
                    out[ih][v] = 0.f;
                }
#pragma unroll
            for (int kx = 0; kx < x; ++kx) {
                uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    uint32_t r[4];
                    ldm(r, ab + (tri(I - 1, J + kx) * NX + pl) * 512);
                    b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                }
                mma_pair<NX, NX, NX>(acc[0], acc[1], y[kx], b0, b1);
            }
            uint32_t a[NX][4], b0[NX][2], b1[NX][2];
            to_a<NX>(acc[0], acc[1], one, one, a);
#pragma unroll
            for (int pl = 0; pl < NX; ++pl) {
                uint32_t r[4];
                ldm(r, ti + sm.ti(I) + pl * 512);
                b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
            }
            mma_pair<NX, NX, NX>(out[0], out[1], a, b0, b1);
            to_a<NX>(out[0], out[1], one, one, y[x]);
#pragma unroll
            for (int pl = 0; pl < NX; ++pl)
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    *reinterpret_cast<uint32_t*>(Y + (pl * kYBlocks + tri(I, J)) * 512 + ((m & 1) * 2 + (m >> 1)) * 128 + lane * 4) =
                        y[x][pl][m];
        }
    }
}

// ------------------------------------------------------------------ the walk
// STATES: a walk for the states alone, without outputs and their operands.
template <typename T, int DP, bool STATES>
struct ChainSmem {
    static constexpr int kIn = kDeltaIn<T>, kX = kDeltaPlanes;
    // chunks in shared memory: the one at work and the next; where it fits, the last one for the output warps, which then
    // finish a chunk while the chain is at the next (8 x 8 heads of 8192 tokens, bf16: 496 us with the gates' kernel and the
    // planes kept, 535 us with a chunk more on its way in that place); where only one fits, it waits for its turn
    static constexpr int kStages = kIn == 1 ? (DP == 64 && !STATES ? 3 : 2) : DP == 64 ? 2 : 1;
    static constexpr bool kLag = kStages == 3;
    struct Stage {
        alignas(128) unsigned char k[kIn * 64 * DP * 2];
        alignas(128) unsigned char q[STATES ? 16 : kIn * 64 * DP * 2];
        alignas(128) unsigned char v[kIn * 64 * kDeltaCols * 2];
        alignas(128) unsigned char y[kX * kYBlocks * 512];
        alignas(128) unsigned char P[STATES ? 16 : kX * kYBlocks * 512];
        Gates s;
    } st[kStages];
    // threads: the chain's 128, the output warps' 128, the loading 128; CTAs per SM
    static constexpr int kThreads = STATES ? 256 : 384, kChain = STATES ? 128 : 256;
    // by pair of warps
    alignas(16) unsigned char S0[2][DP / 16][kX * 512];  // S^T before the chunk, planes
    alignas(16) unsigned char R[2][4][kX * 512];         // -(beta R)^T, planes
    // W^T for the update and the outputs. 16-bit inputs: planes of beta W and of e^{g_C - g} beta W (and of W where
    // it is kept), converted once by the warp that has it. float32 inputs (no room), and the states' pass (two CTAs
    // share an SM without): W, converted by each reader
    static constexpr bool kShared = kIn < 3 && !STATES;
    alignas(16) unsigned char Wb[kLag ? 2 : 1][2][kShared ? 4 : 1][kX * 512];  // (by chunk parity where outputs lag)
    alignas(16) unsigned char Wk[2][kShared ? 4 : 1][kX * 512];
    union {
        float4 W[2][kShared ? 1 : 8 * 32];
        unsigned char Wp[2][STATES ? 1 : 4][kX * 512];
    } w;
    // outputs on their way to memory: in the place of Y, which nobody reads any more by then
    static constexpr int kOutPitch = 16 * sizeof(T) + 16;
    static_assert(4 * 32 * kOutPitch <= kX * kYBlocks * 512, "staged outputs");
};

// One warp of a chain pair: half `A` of d of S^T in its accumulators; R and W of its token blocks.
template <typename T, int DP, bool OUT, bool KEEP>
__device__ __forceinline__ void chain_warp(ChainSmem<T, DP, !OUT && !KEEP>& sm, const DeltaParams& p, const WalkJob& job, int A, int pair, int lane) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes, NST = ChainSmem<T, DP, !OUT && !KEEP>::kStages;
    constexpr int NH = DP / 16;  // 8-column blocks of half of d
    constexpr bool kShared = ChainSmem<T, DP, !OUT && !KEEP>::kShared;
    const int g = lane >> 2, t = lane & 3;
    const Own own(A);
    const float2 one = make_float2(1.f, 1.f);
    float S[NH][4];
    const int col0 = job.c0 + 16 * pair;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 8 * (A * NH + n) + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
            S[n][i] = job.ident ? (d == col ? 1.f : 0.f) : (job.in && d < p.d && col < job.ld) ? job.in[(int64_t)d * job.ld + col] : 0.f;
        }
    auto put_state = [&]() {
#pragma unroll
        for (int kk = 0; kk < NH / 2; ++kk) {
            uint32_t a[NX][4];
            to_a<NX>(S[2 * kk], S[2 * kk + 1], one, one, a);
            put_a<NX>(sm.S0[pair][A * (NH / 2) + kk], a, lane);
        }
    };
    put_state();
    __syncthreads();
    for (int c = job.begin; c < job.end; ++c) {
        if (NST == 1) __syncthreads();  // the chunk is loaded
        auto& st = sm.st[c % NST];
        const Gates& s = st.s;
        if (s.any) {
            const uint32_t kt = smem_addr(st.k), vt = smem_addr(st.v), yt = smem_addr(st.y) + lane * 16;
            float W[4][4];  // (K S0)^T, then R^T, then W^T: blocks 2 u + half of this warp's tokens
            zero_acc<4>(W);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a[NX][4];
                get_a<NX>(a, sm.S0[pair][kk], lane);
                mma_rows<DP, NX, NIN, NX>(W, a, kt, 16 * own.b0, 16 * own.b1, kk, lane);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // R = V - e^g K S0; -beta R for both warps
                const int tok = 16 * own.at(u) + 2 * t;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int pl = 0; pl < NIN; ++pl) {
                    uint32_t r[4];
                    a_cols<kDeltaCols>(r, vt + pl * (64 * kDeltaCols * 2), 16 * own.at(u), pair, lane);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const float2 x = unpack_bf16(r[m]);
                        v[2 * m] += x.x;
                        v[2 * m + 1] += x.y;
                    }
                }
                float2 be[2];
#pragma unroll
                for (int jh = 0; jh < 2; ++jh) {
                    const float2 eg = *reinterpret_cast<const float2*>(&s.eg[tok + 8 * jh]);
                    be[jh] = *reinterpret_cast<const float2*>(&s.beta[tok + 8 * jh]);
                    be[jh] = make_float2(-be[jh].x, -be[jh].y);
                    float(&w)[4] = W[2 * u + jh];
                    w[0] = fmaf(-eg.x, w[0], v[4 * jh]);
                    w[1] = fmaf(-eg.y, w[1], v[4 * jh + 1]);
                    w[2] = fmaf(-eg.x, w[2], v[4 * jh + 2]);
                    w[3] = fmaf(-eg.y, w[3], v[4 * jh + 3]);
                }
                uint32_t a[NX][4];
                to_a<NX>(W[2 * u], W[2 * u + 1], be[0], be[1], a);
                put_a<NX>(sm.R[pair][own.at(u)], a, lane);
            }
            bar_sync(4 + pair, 64);
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {  // W^T = R^T - (beta R)^T Y^T
                if (jb > own.b1) break;
                uint32_t a[NX][4];
                get_a<NX>(a, sm.R[pair][jb], lane);
                mma_blocks<NX, NX, true>(W, a, jb <= own.b0, yt + tri(own.b0, jb) * 512, true, yt + tri(own.b1, jb) * 512);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int jb = own.at(u);
                if constexpr (kShared) {
                    float2 fb[2], fk[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 kd = *reinterpret_cast<const float2*>(&s.kd[16 * jb + 8 * i + 2 * t]);
                        fb[i] = *reinterpret_cast<const float2*>(&s.beta[16 * jb + 8 * i + 2 * t]);
                        fk[i] = make_float2(fb[i].x * kd.x, fb[i].y * kd.y);
                    }
                    uint32_t a[NX][4];
                    to_a<NX>(W[2 * u], W[2 * u + 1], fk[0], fk[1], a);
                    put_a<NX>(sm.Wk[pair][jb], a, lane);
                    if (OUT) {
                        to_a<NX>(W[2 * u], W[2 * u + 1], fb[0], fb[1], a);
                        put_a<NX>(sm.Wb[ChainSmem<T, DP, !OUT && !KEEP>::kLag ? c & 1 : 0][pair][jb], a, lane);
                    }
                    if (KEEP) {
                        to_a<NX>(W[2 * u], W[2 * u + 1], one, one, a);
                        put_a<NX>(sm.w.Wp[pair][jb], a, lane);
                    }
                } else {
                    sm.w.W[pair][2 * jb * 32 + lane] = as_float4(W[2 * u]);
                    sm.w.W[pair][(2 * jb + 1) * 32 + lane] = as_float4(W[2 * u + 1]);
                }
            }
            float U[NH][4];  // the chunk's update, summed by itself (see mma_set) and added to the state once, rounded
            zero_acc<NH>(U);
            bar_sync(1, ChainSmem<T, DP, !OUT && !KEEP>::kChain);  // W is there for both pairs and the output warps, which have read S0
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {  // S'^T = e^{g_C} S0^T + (e^{g_C - g} beta W)^T K over this half of d
                uint32_t a[NX][4];
                if constexpr (kShared) {
                    get_a<NX>(a, sm.Wk[pair][jb], lane);
                } else {
                    float w0[4], w1[4];
                    get_acc2(w0, w1, sm.w.W[pair] + 2 * jb * 32, lane);
                    float2 f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 16 * jb + 8 * i + 2 * t;
                        const float2 be = *reinterpret_cast<const float2*>(&s.beta[j]), kd = *reinterpret_cast<const float2*>(&s.kd[j]);
                        f[i] = make_float2(be.x * kd.x, be.y * kd.y);
                    }
                    to_a<NX>(w0, w1, f[0], f[1], a);
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

// One warp of an output pair: the outputs of 16 columns for its token blocks, and its share of the planes.
template <typename T, int DP, bool OUT, bool KEEP>
__device__ __forceinline__ void output_warp(ChainSmem<T, DP, !OUT && !KEEP>& sm, const DeltaParams& p, const WalkJob& job, int A, int pair, int lane) {
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes, NST = ChainSmem<T, DP, !OUT && !KEEP>::kStages;
    const int g = lane >> 2, t = lane & 3;
    const Own own(A);
    const float2 one = make_float2(1.f, 1.f);
    const int64_t bh = job.bh;
    const int cb = job.cb, ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    T* o = OUT ? static_cast<T*>(p.o.p) + tensor_base(p.o, job.b, job.h) : nullptr;
    constexpr bool kShared = ChainSmem<T, DP, !OUT && !KEEP>::kShared;
    constexpr int kPitch = ChainSmem<T, DP, !OUT && !KEEP>::kOutPitch, kPieces = 16 * sizeof(T) / 16;  // bytes of a staged row, its 16-byte pieces
    const int col0 = cb * kDeltaCols + 16 * pair, width = min(16, p.e - col0);
    const bool whole = OUT && p.o.vec && width == 16;
    constexpr bool kLag = ChainSmem<T, DP, !OUT && !KEEP>::kLag;
    float O[4][4];  // blocks 2 u + half of this warp's tokens
    auto planes_of_w = [&](int c) {
        const int64_t cw = (bh * p.nc + c) * 2 * ncb + 2 * cb + pair;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int jb = own.at(u);
            uint32_t a[NX][4];
            if constexpr (kShared) {
                get_a<NX>(a, sm.w.Wp[pair][jb], lane);
            } else {
                float w0[4], w1[4];
                get_acc2(w0, w1, sm.w.W[pair] + 2 * jb * 32, lane);
                to_a<NX>(w0, w1, one, one, a);
            }
            store_matrices<NX>(p.W + (cw * 4 + jb) * (NX * 512), a, lane);
        }
    };
    auto finish = [&](int c) {  // the scores' part of the outputs of chunk c, and the outputs to memory
        auto& st = sm.st[c % NST];
        const Gates& s = st.s;
        const int n0 = c * kDeltaC;
        unsigned char* stage = st.y + (2 * pair + A) * (32 * kPitch);
        const bool any = s.any;
        if (any) {
            const uint32_t pt = smem_addr(st.P) + lane * 16;
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {
                if (jb > own.b1) break;
                uint32_t a[NX][4];
                if constexpr (kShared) {
                    get_a<NX>(a, sm.Wb[kLag ? c & 1 : 0][pair][jb], lane);
                } else {
                    float w0[4], w1[4];
                    get_acc2(w0, w1, sm.w.W[pair] + 2 * jb * 32, lane);
                    to_a<NX>(w0, w1, *reinterpret_cast<const float2*>(&s.beta[16 * jb + 2 * t]),
                             *reinterpret_cast<const float2*>(&s.beta[16 * jb + 8 + 2 * t]), a);
                }
                mma_blocks<NX, NX, false>(O, a, jb <= own.b0, pt + tri(own.b0, jb) * 512, true, pt + tri(own.b1, jb) * 512);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {  // staged rows: 16 u + 8 half + ..
                T* r0 = reinterpret_cast<T*>(stage + (8 * n + 2 * t) * kPitch);
                T* r1 = reinterpret_cast<T*>(stage + (8 * n + 2 * t + 1) * kPitch);
                r0[g] = from_f<T>(O[n][0]);
                r1[g] = from_f<T>(O[n][1]);
                r0[g + 8] = from_f<T>(O[n][2]);
                r1[g + 8] = from_f<T>(O[n][3]);
            }
            __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int i = lane + 32 * x, row = i / kPieces, piece = i % kPieces;
            const int tok = 16 * own.at(row >> 4) + (row & 15);
            if (n0 + tok >= p.N) continue;
            T* dst = o + (n0 + tok) * p.o.sn + col0;
            const bool live = any && s.live[tok];
            const unsigned char* src = stage + row * kPitch + piece * 16;
            if (whole) {
                reinterpret_cast<uint4*>(dst)[piece] = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
            } else {
                constexpr int kPer = 16 / sizeof(T);
#pragma unroll
                for (int y = 0; y < kPer; ++y)
                    if (piece * kPer + y < width)
                        dst[piece * kPer + y] = live ? reinterpret_cast<const T*>(src)[y] : from_f<T>(0.f);
            }
        }
    };
    __syncthreads();
    for (int c = job.begin; c < job.end; ++c) {
        if (NST == 1) __syncthreads();
        if (OUT && kLag && c > job.begin) finish(c - 1);
        auto& st = sm.st[c % NST];
        const Gates& s = st.s;
        if (s.any) {
            const uint32_t qt = smem_addr(st.q);
            const int64_t cw = (bh * p.nc + c) * 2 * ncb + 2 * cb + pair;  // chunk and group of 16 columns
            zero_acc<4>(O);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {  // (Q S0)^T
                if (!OUT && kk % 2 != A) continue;
                uint32_t a[NX][4];
                get_a<NX>(a, sm.S0[pair][kk], lane);
                if (KEEP && kk % 2 == A) store_matrices<NX>(p.S0 + (cw * (DP / 16) + kk) * (NX * 512), a, lane);
                if (OUT) mma_rows<DP, NX, NIN, NX>(O, a, qt, 16 * own.b0, 16 * own.b1, kk, lane);
            }
            if (OUT) {
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float2 eg = *reinterpret_cast<const float2*>(&s.eg[16 * own.at(n >> 1) + 8 * (n & 1) + 2 * t]);
                    O[n][0] *= p.scale * eg.x;
                    O[n][1] *= p.scale * eg.y;
                    O[n][2] *= p.scale * eg.x;
                    O[n][3] *= p.scale * eg.y;
                }
            }
            bar_sync(1, 256);
            if (KEEP) planes_of_w(c);
        }
        if (OUT && !kLag) finish(c);
        __syncthreads();
    }
    if (OUT && kLag) finish(job.end - 1);
}

// OUT: writes o. KEEP: writes the planes of S0 and W that the backward reads.
// Neither: the states alone, in half the shared memory, so that two CTAs share an SM.
template <typename T, int DP, bool STATES>
constexpr int chain_ctas() {
    return STATES && sizeof(ChainSmem<T, DP, STATES>) <= 112 * 1024 ? 2 : 1;
}

template <typename T, int DP, bool OUT, bool KEEP>
__global__ void __launch_bounds__(ChainSmem<T, DP, !OUT && !KEEP>::kThreads, chain_ctas<T, DP, !OUT && !KEEP>())
delta_chain_kernel(const DeltaParams p) {
    constexpr bool kStates = !OUT && !KEEP;
    constexpr int NIN = kDeltaIn<T>, NX = kDeltaPlanes;
    constexpr int NST = ChainSmem<T, DP, kStates>::kStages;
    extern __shared__ __align__(128) unsigned char raw[];
    using Smem = ChainSmem<T, DP, kStates>;
    Smem& sm = *reinterpret_cast<Smem*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // (sequence, segment, block of columns), the last fastest. States only: the first nseg - 1 segments, with the
    // identity's columns after the value columns, but for the first segment (nobody asks what it does to a state)
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols, ndb = kStates ? (p.d + kDeltaCols - 1) / kDeltaCols : 0, ncols = ncb + ndb;
    const int nseg = kStates ? p.nseg - 1 : p.nseg;
    const unsigned per_seq = (unsigned)(nseg * ncols - ndb), bh32 = blockIdx.x / per_seq;
    const int at = (int)(blockIdx.x - bh32 * per_seq) + ndb;  // (the first segment's columns at ndb ..)
    const int seg = at / ncols, col = at - seg * ncols;
    WalkJob job;
    job.bh = bh32;
    job.b = (int)(bh32 / (unsigned)p.H);
    job.h = (int)(bh32 - job.b * (unsigned)p.H);
    job.ident = kStates && col < ndb;
    job.cb = job.ident ? col : col - ndb;
    job.c0 = job.cb * kDeltaCols;
    job.begin = seg * p.seg_chunks;
    job.end = min(p.nc, job.begin + p.seg_chunks);
    job.ld = job.ident ? DP : p.e;
    job.rows = job.ident ? DP : p.d;
    const int64_t before = job.bh * (p.nseg - 1) + seg;  // the segment's slot in seg_S and seg_M
    if (kStates) {
        job.in = seg == 0 && !job.ident && p.S_in ? p.S_in + job.bh * p.d * p.e : nullptr;
        job.out = job.ident ? p.seg_M + before * (DP * DP) : p.seg_S + before * p.d * p.e;
    } else {
        const float* S_in = p.seg_in ? p.seg_in : p.S_in;
        job.in = seg ? p.seg_S + (before - 1) * p.d * p.e : S_in ? S_in + job.bh * p.d * p.e : nullptr;
        job.out = seg + 1 == nseg && p.S_out ? p.S_out + job.bh * p.d * p.e : nullptr;
    }
    if (warp < 4) {
        chain_warp<T, DP, OUT, KEEP>(sm, p, job, warp & 1, warp >> 1, lane);
    } else if (!kStates && warp < 8) {
        if constexpr (!kStates) output_warp<T, DP, OUT, KEEP>(sm, p, job, warp & 1, (warp >> 1) & 1, lane);
    } else {  // ---------------------------------------------------------- loads
        // the loads of a chunk are in flight for a whole iteration or two
        const int lt = tid - Smem::kChain;
        const int64_t bh = job.bh;
        const int b = job.b, h = job.h, begin = job.begin, end = job.end, c0 = job.c0;
        const Gates* gates = p.gates + bh * p.nc;
        const int64_t kb = tensor_base(p.k, b, h), qb = tensor_base(p.q, b, h), vb = tensor_base(p.v, b, h);
        if (job.ident) {  // V is 0 in every stage
            for (int i = 0; i < NST; ++i)
                for (int x = lt * 16; x < (int)sizeof(sm.st[i].v); x += 128 * 16)
                    *reinterpret_cast<uint4*>(sm.st[i].v + x) = make_uint4(0, 0, 0, 0);
        }
        constexpr int kMat = NX * kYBlocks * 512;
        const unsigned char* Y = p.Y + bh * p.nc * kMat;
        const unsigned char* P = p.P + bh * p.nc * kMat;
        bool async = false;
        if constexpr (NIN == 1) async = p.k.vec && p.q.vec && p.v.vec && p.d % 8 == 0 && p.e % 8 == 0;
        if (async) {
            // bf16: asynchronous copies, chunk c + 1's while c is computed (8 x 12 heads of 2047 tokens: 229 us with the
            // gates' kernel and rows on 16 bytes, 367 us through registers, element by element, without)
            int any_next = gates[begin].any;
            auto start = [&](int c) {
                if (c < end) {
                    const int any = any_next;
                    any_next = c + 1 < end ? gates[c + 1].any : 0;
                    auto& st = sm.st[c % NST];
                    async16<128>(reinterpret_cast<unsigned char*>(&st.s), reinterpret_cast<const unsigned char*>(gates + c), sizeof(Gates), lt);
                    if (any) {
                        const int n0 = c * kDeltaC;
                        async_tile<T, DP, 128>(st.k, p.k, kb, n0, 0, p.d, p.N, lt);
                        if (!job.ident) async_tile<T, kDeltaCols, 128>(st.v, p.v, vb, n0, c0, p.e, p.N, lt);
                        async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                        if constexpr (OUT) {
                            async_tile<T, DP, 128>(st.q, p.q, qb, n0, 0, p.d, p.N, lt);
                            async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                        }
                    }
                }
            };
            auto finish = [&](int c) {
                async_wait();
                if (c >= end) return;
                bar_sync(3, 128);
                auto& st = sm.st[c % NST];
                if (st.s.any && !st.s.full) {
                    clear_dead<DP, 128>(st.k, st.s.live, lt);
                    if constexpr (OUT) clear_dead<DP, 128>(st.q, st.s.live, lt);
                    clear_dead<kDeltaCols, 128>(st.v, st.s.live, lt);
                }
            };
            start(begin);
            finish(begin);
            __syncthreads();
            for (int c = begin; c < end; ++c) {
                start(c + 1);
                finish(c + 1);
                __syncthreads();
            }
        } else {
            if constexpr (NST == 1) {  // (no room for a second chunk: each tile is loaded when its turn comes)
                __syncthreads();
                for (int c = begin; c < end; ++c) {
                    auto& st = sm.st[0];
                    copy16<128>(reinterpret_cast<unsigned char*>(&st.s), reinterpret_cast<const unsigned char*>(gates + c), sizeof(Gates), lt);
                    bar_sync(3, 128);
                    if (st.s.any) {
                        const int n0 = c * kDeltaC;
                        load_tile<T, DP, NIN, 128>(st.k, p.k, kb, n0, 0, p.d, p.N, st.s.live, lt);
                        if (!job.ident) load_tile<T, kDeltaCols, NIN, 128>(st.v, p.v, vb, n0, c0, p.e, p.N, st.s.live, lt);
                        async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                        if constexpr (OUT) {
                            load_tile<T, DP, NIN, 128>(st.q, p.q, qb, n0, 0, p.d, p.N, st.s.live, lt);
                            async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                        }
                        async_wait();
                    }
                    __syncthreads();
                    __syncthreads();
                }
            } else {
                TileRegs<T, DP, 128> k, q;
                TileRegs<T, kDeltaCols, 128> v;
                ByteRegs<sizeof(Gates), 128> s;
                int any = 0, any_next = gates[begin].any;  // of the chunk in the registers, and of the one after it
                auto issue = [&](int c) {
                    any = any_next;
                    any_next = c + 1 < end ? gates[c + 1].any : 0;
                    if (c >= end) return;
                    s.issue(gates + c, lt);
                    if (!any) return;
                    const int n0 = c * kDeltaC;
                    k.issue(p.k, kb, n0, 0, p.d, p.N, lt);
                    if (!job.ident) v.issue(p.v, vb, n0, c0, p.e, p.N, lt);
                    if constexpr (OUT) {
                        q.issue(p.q, qb, n0, 0, p.d, p.N, lt);
                    }
                };
                auto store = [&](int c) {
                    if (c >= end) return;
                    auto& st = sm.st[c % NST];
                    s.store(&st.s, lt);
                    bar_sync(3, 128);
                    if (!any) return;
                    async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                    if constexpr (OUT) async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                    k.template store_planes<NIN>(st.k, st.s.live, lt);
                    if (!job.ident) v.template store_planes<NIN>(st.v, st.s.live, lt);
                    if constexpr (OUT) {
                        q.template store_planes<NIN>(st.q, st.s.live, lt);
                    }
                };
                issue(begin);
                store(begin);
                issue(begin + 1);
                async_wait();
                __syncthreads();
                for (int c = begin; c < end; ++c) {
                    store(c + 1);
                    issue(c + 2);
                    async_wait();
                    __syncthreads();
                }
            }
        }
    }
}

template <typename T, int DP>
cudaError_t chain_t(const DeltaParams& p, cudaStream_t st) {
    using Walk = ChainSmem<T, DP, false>;
    using States = ChainSmem<T, DP, true>;
    static_assert(sizeof(Walk) <= 227 * 1024 && sizeof(States) <= 227 * 1024, "shared memory");
    const int64_t bh = (int64_t)p.B * p.H, ncb = (p.e + kDeltaCols - 1) / kDeltaCols, ndb = (p.d + kDeltaCols - 1) / kDeltaCols;
    auto run = [&](auto kernel, int64_t blocks, int threads = Walk::kThreads, size_t smem = sizeof(Walk)) {
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
        kernel<<<(unsigned)blocks, threads, smem, st>>>(p);
        return cudaGetLastError();
    };
    if (p.nseg > 1) {
        cudaError_t err = run(delta_chain_kernel<T, DP, false, false>, bh * ((p.nseg - 1) * (ncb + ndb) - ndb), States::kThreads, sizeof(States));
        if (err != cudaSuccess) return err;
        if ((err = join_t<DP>(p, st)) != cudaSuccess) return err;
    }
    if (!p.o.p) return run(delta_chain_kernel<T, DP, false, true>, bh * p.nseg * ncb);
    if (p.S0) return run(delta_chain_kernel<T, DP, true, true>, bh * p.nseg * ncb);
    return run(delta_chain_kernel<T, DP, true, false>, bh * p.nseg * ncb);
}

template <typename T, int DP>
cudaError_t fwd_t(const DeltaParams& p, cudaStream_t st) {
    const size_t prep = sizeof(PrepSmem<T, DP>);
    cudaError_t err = cudaFuncSetAttribute(delta_prep_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prep);
    if (err != cudaSuccess) return err;
    delta_prep_kernel<T, DP><<<(unsigned)((int64_t)p.B * p.H * p.nc), 128, prep, st>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    return chain_t<T, DP>(p, st);
}

}  // namespace
}  // namespace subq
