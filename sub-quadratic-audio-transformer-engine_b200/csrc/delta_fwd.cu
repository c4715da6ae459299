// Chunked forward of the gated delta rule (see delta_common.cuh for the algebra).
//
// delta_prep_kernel: gates, Y and scores of every chunk, all chunks at once.
// delta_chain_kernel: the walk over the chunks. A warp owns 16 value columns of
// one sequence and keeps S^T [16 x d] in its accumulators: the m16n8k16
// accumulator layout is the A operand layout of the next product, so the chain
// S0 -> R -> W -> S' stays in one warp's registers and no warp waits for another
// value column. All products are transposed accordingly (rows = value columns,
// columns = tokens or d). Per CTA, 32 columns: two such chain warps; two output
// warps (Q S0 and score W products of the chain warp with the same columns, from
// the float32 S0 and W it leaves in shared memory; they also write the planes the
// backward reads); and four warps that load the next chunks. The chain warp does
// nothing that another warp can do.
#include "delta_common.cuh"
#include "delta_launch.h"
#include "scan_launch.h"

namespace subq {
namespace {

using namespace dl;

// ------------------------------------------------------------------ gates, Y and scores per chunk
template <typename T, int DP>
struct PrepSmem {
    static constexpr int kIn = DeltaType<T>::kIn, kX = DeltaType<T>::kX;
    Gates s;
    alignas(16) float A[kDeltaC][kDeltaC + 4];
    alignas(128) unsigned char Ab[6 * kX * 512];  // -A_IK beta, blocks I > K: [block][plane]
    alignas(128) unsigned char Ti[4 * kX * 512];  // (I + A_II beta)^-1
    alignas(128) unsigned char k[kIn * 64 * DP * 2];
    alignas(128) unsigned char q[kIn * 64 * DP * 2];
};

// Y by 16 x 16 blocks. With T_I = (I + A_II beta)^-1 (forward substitution, a
// column per lane), block column J of Y is one warp's:
//   Y_JJ^T = A_JJ^T T_J^T,   Y_IJ^T = (A_IJ^T - sum_{J <= K < I} Y_KJ^T (A_IK beta)^T) T_I^T,
// transposed so that each result is, in its registers, the A operand of the next product.
template <typename T, int DP>
__global__ void __launch_bounds__(128) delta_prep_kernel(const DeltaParams p) {
    constexpr int NIN = DeltaType<T>::kIn, NX = DeltaType<T>::kX, kTile = 64 * DP * 2;
    extern __shared__ __align__(128) unsigned char raw[];
    PrepSmem<T, DP>& sm = *reinterpret_cast<PrepSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int64_t chunk = blockIdx.x;  // bh * nc + c
    const int64_t bh = chunk / p.nc;
    const int c = (int)(chunk % p.nc), b = (int)(bh / p.H), h = (int)(bh % p.H), n0 = c * kDeltaC;
    {
        TileRegs<T, DP, 128> k, q;
        k.issue(p.k, tensor_base(p.k, b, h), n0, 0, p.d, p.N, tid);
        if (p.P) q.issue(p.q, tensor_base(p.q, b, h), n0, 0, p.d, p.N, tid);
        if (warp == 0) form_gates(sm.s, p, b, h, n0, lane);
        __syncthreads();
        copy16<128>(reinterpret_cast<unsigned char*>(p.gates + chunk), reinterpret_cast<const unsigned char*>(&sm.s), sizeof(Gates), tid);
        if (!sm.s.any) return;  // nothing else of a dead chunk is read
        k.template store_planes<NIN>(sm.k, sm.s.live, tid);
        if (p.P) q.template store_planes<NIN>(sm.q, sm.s.live, tid);
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
                    mma_planes<NIN, NIN, NX>(acc[2 * jb], a, b0);
                    mma_planes<NIN, NIN, NX>(acc[2 * jb + 1], a, b1);
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
                    *reinterpret_cast<float2*>(&sm.A[i][j]) = make_float2(x, y);
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
    if (p.P)
        score_rows<DP, NIN, NX>(p.P + chunk * (NX * kYBlocks * 512), smem_addr(sm.q), smem_addr(sm.k), sm.s, p.scale, 3 - warp, lane);
    __syncwarp();  // the diagonal block is this warp's own
    {
        const int col = lane & 15, r0 = 16 * warp;
        float ti[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // T e_col: t_i = delta - sum_j A_ij beta_j t_j, kept as beta_j t_j
            float x = i == col ? 1.f : 0.f, y = 0.f;
#pragma unroll
            for (int j = 0; j < i; j += 2) {
                const float2 a = *reinterpret_cast<const float2*>(&sm.A[r0 + i][r0 + j]);
                x = fmaf(-a.x, ti[j], x);
                if (j + 1 < i) y = fmaf(-a.y, ti[j + 1], y);
            }
            x += y;
            if (lane < 16) {
                unsigned char* at = sm.Ti + warp * (NX * 512) + ((i >> 3) * 2 + (col >> 3)) * 128 + (i & 7) * 16 + (col & 7) * 2;
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
        const uint32_t ab = smem_addr(sm.Ab) + lane * 16, ti = smem_addr(sm.Ti) + lane * 16;
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
                    acc[ih][v] = sm.A[16 * I + 8 * ih + 2 * t + (v & 1)][16 * J + g + 8 * (v >> 1)];
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
                mma_planes<NX, NX, NX>(acc[0], y[kx], b0);
                mma_planes<NX, NX, NX>(acc[1], y[kx], b1);
            }
            uint32_t a[NX][4], b0[NX][2], b1[NX][2];
            to_a<NX>(acc[0], acc[1], one, one, a);
#pragma unroll
            for (int pl = 0; pl < NX; ++pl) {
                uint32_t r[4];
                ldm(r, ti + (I * NX + pl) * 512);
                b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
            }
            mma_planes<NX, NX, NX>(out[0], a, b0);
            mma_planes<NX, NX, NX>(out[1], a, b1);
            to_a<NX>(out[0], out[1], one, one, y[x]);
#pragma unroll
            for (int pl = 0; pl < NX; ++pl)
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    *reinterpret_cast<uint32_t*>(Y + (pl * kYBlocks + tri(I, J)) * 512 + m * 128 + lane * 4) = y[x][pl][m];
        }
    }
}

// ------------------------------------------------------------------ the walk
template <typename T, int DP>
struct ChainSmem {
    static constexpr int kIn = DeltaType<T>::kIn, kX = DeltaType<T>::kX;
    // chunks in shared memory: the one at work, the next, and for bf16 one on its way; one where two do not fit
    static constexpr int kStages = kIn == 1 ? 3 : DP == 64 ? 2 : 1;
    struct Stage {
        alignas(128) unsigned char k[kIn * 64 * DP * 2];
        alignas(128) unsigned char q[kIn * 64 * DP * 2];
        alignas(128) unsigned char v[kIn * 64 * kDeltaCols * 2];
        alignas(128) unsigned char y[kX * kYBlocks * 512];
        alignas(128) unsigned char P[kX * kYBlocks * 512];
        Gates s;
    } st[kStages];
    float4 S0[2][2][DP / 8 * 32];  // S^T accumulators before the chunk: [chunk parity][chain warp]
    float4 W[2][8 * 32];           // W^T accumulators
    alignas(16) unsigned char out[2][kDeltaC * (16 * sizeof(T) + 16)];
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, 1) delta_chain_kernel(const DeltaParams p) {
    constexpr int NIN = DeltaType<T>::kIn, NX = DeltaType<T>::kX, kTile = 64 * DP * 2;
    constexpr int NST = ChainSmem<T, DP>::kStages;
    extern __shared__ __align__(128) unsigned char raw[];
    ChainSmem<T, DP>& sm = *reinterpret_cast<ChainSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    const int64_t bh = blockIdx.x / ncb;
    const int cb = blockIdx.x % ncb, b = (int)(bh / p.H), h = (int)(bh % p.H), c0 = cb * kDeltaCols;
    const int g = lane >> 2, t = lane & 3;

    if (warp < 2) {  // ---------------------------------------------------- chain
        float S[DP / 8][4];
        const int col0 = c0 + 16 * warp;
        const float* S_in = p.S_in ? p.S_in + bh * p.d * p.e : nullptr;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 8 * n + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
                S[n][i] = (S_in && d < p.d && col < p.e) ? S_in[(int64_t)d * p.e + col] : 0.f;
            }
        put_acc<DP / 8>(sm.S0[0][warp], S, lane);
        __syncthreads();
        for (int c = 0; c < p.nc; ++c) {
            if (NST == 1) __syncthreads();  // the chunk is loaded
            auto& st = sm.st[c % NST];
            const Gates& s = st.s;
            if (s.any) {
                const uint32_t kt = smem_addr(st.k);
                const float2 one = make_float2(1.f, 1.f);
                float X[8][4];
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) X[n][i] = 0.f;
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {  // X = S0^T K^T
                    uint32_t a[NX][4];
                    to_a<NX>(S[2 * kk], S[2 * kk + 1], one, one, a);
#pragma unroll
                    for (int jp = 0; jp < 4; ++jp) {
                        uint32_t b0[NIN][2], b1[NIN][2];
#pragma unroll
                        for (int pl = 0; pl < NIN; ++pl) {
                            uint32_t r[4];
                            b_rows<DP>(r, kt + pl * kTile, 16 * jp, kk, lane);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NIN, NX>(X[2 * jp], a, b0);
                        mma_planes<NX, NIN, NX>(X[2 * jp + 1], a, b1);
                    }
                }
                // R = V - e^g X, and -beta R as the operand
                uint32_t ra[4][NX][4];
                const uint32_t vt = smem_addr(st.v);
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) {
                        uint32_t r[4];
                        a_cols<kDeltaCols>(r, vt + pl * (64 * kDeltaCols * 2), 16 * jb, warp, lane);
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const float2 x = unpack_bf16(r[m]);
                            v[2 * m] += x.x;
                            v[2 * m + 1] += x.y;
                        }
                    }
#pragma unroll
                    for (int jh = 0; jh < 2; ++jh) {
                        const float2 eg = *reinterpret_cast<const float2*>(&s.eg[16 * jb + 8 * jh + 2 * t]);
                        float(&x)[4] = X[2 * jb + jh];
                        x[0] = fmaf(-eg.x, x[0], v[4 * jh]);
                        x[1] = fmaf(-eg.y, x[1], v[4 * jh + 1]);
                        x[2] = fmaf(-eg.x, x[2], v[4 * jh + 2]);
                        x[3] = fmaf(-eg.y, x[3], v[4 * jh + 3]);
                    }
                    const float2 b0 = *reinterpret_cast<const float2*>(&s.beta[16 * jb + 2 * t]);
                    const float2 b1 = *reinterpret_cast<const float2*>(&s.beta[16 * jb + 8 + 2 * t]);
                    to_a<NX>(X[2 * jb], X[2 * jb + 1], make_float2(-b0.x, -b0.y), make_float2(-b1.x, -b1.y), ra[jb]);
                }
                // W^T = R^T - (beta R)^T Y^T
                const uint32_t yt = smem_addr(st.y) + lane * 16;
#pragma unroll
                for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                    for (int jb = 0; jb <= ib; ++jb) {
                        uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) {
                            uint32_t r[4];
                            ldm_t(r, yt + pl * (kYBlocks * 512) + tri(ib, jb) * 512);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NX, NX>(X[2 * ib], ra[jb], b0);
                        mma_planes<NX, NX, NX>(X[2 * ib + 1], ra[jb], b1);
                    }
                put_acc<8>(sm.W[warp], X, lane);
                bar_arrive(1, 128);
                // S'^T = e^{g_C} S0^T + (e^{g_C - g} beta W)^T K
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[n][i] *= s.eC;
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    uint32_t a[NX][4];
                    float2 f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 16 * jb + 8 * i + 2 * t;
                        f[i] = make_float2(s.beta[j] * s.kd[j], s.beta[j + 1] * s.kd[j + 1]);
                    }
                    to_a<NX>(X[2 * jb], X[2 * jb + 1], f[0], f[1], a);
#pragma unroll
                    for (int np = 0; np < DP / 16; ++np) {
                        uint32_t b0[NIN][2], b1[NIN][2];
#pragma unroll
                        for (int pl = 0; pl < NIN; ++pl) {
                            uint32_t r[4];
                            b_cols<DP>(r, kt + pl * kTile, 16 * jb, np, lane);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NIN, NX>(S[2 * np], a, b0);
                        mma_planes<NX, NIN, NX>(S[2 * np + 1], a, b1);
                    }
                }
            } else {
                bar_arrive(1, 128);
            }
            put_acc<DP / 8>(sm.S0[(c + 1) & 1][warp], S, lane);
            __syncthreads();
        }
        if (p.S_out) {
            float* S_out = p.S_out + bh * p.d * p.e;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 8 * n + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
                    if (d < p.d && col < p.e) S_out[(int64_t)d * p.e + col] = S[n][i];
                }
        }
    } else if (warp < 4) {  // -------------------------------------------- outputs
        const int w = warp - 2;
        T* o = p.o.p ? static_cast<T*>(p.o.p) + tensor_base(p.o, b, h) : nullptr;  // null: states and W only
        constexpr int kPitch = 16 * sizeof(T) + 16;
        __syncthreads();
        for (int c = 0; c < p.nc; ++c) {
            if (NST == 1) __syncthreads();  // the chunk is loaded
            auto& st = sm.st[c % NST];
            const Gates& s = st.s;
            const int n0 = c * kDeltaC, rows = min(kDeltaC, p.N - n0);
            unsigned char* stage = sm.out[w];
            if (s.any) {
                const uint32_t qt = smem_addr(st.q), pt = smem_addr(st.P) + lane * 16;
                const int64_t cw = (bh * p.nc + c) * 2 * ncb + 2 * cb + w;  // chunk and group of 16 columns
                unsigned char* s0dst = p.S0 ? p.S0 + cw * (DP / 16 * NX * 512) : nullptr;
                unsigned char* wdst = p.W ? p.W + cw * (4 * NX * 512) : nullptr;
                float O[8][4];
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) O[n][i] = 0.f;
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {  // S0^T Q^T
                    uint32_t a[NX][4];
                    get_a<NX>(sm.S0[c & 1][w], kk, a, s0dst, lane);
                    if (!o) continue;
#pragma unroll
                    for (int jp = 0; jp < 4; ++jp) {
                        uint32_t b0[NIN][2], b1[NIN][2];
#pragma unroll
                        for (int pl = 0; pl < NIN; ++pl) {
                            uint32_t r[4];
                            b_rows<DP>(r, qt + pl * kTile, 16 * jp, kk, lane);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NIN, NX>(O[2 * jp], a, b0);
                        mma_planes<NX, NIN, NX>(O[2 * jp + 1], a, b1);
                    }
                }
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const float2 eg = *reinterpret_cast<const float2*>(&s.eg[8 * n + 2 * t]);
                    O[n][0] *= p.scale * eg.x;
                    O[n][1] *= p.scale * eg.y;
                    O[n][2] *= p.scale * eg.x;
                    O[n][3] *= p.scale * eg.y;
                }
                bar_sync(1, 128);  // both chain warps' W
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    uint32_t a[NX][4];
                    get_a<NX>(sm.W[w], jb, a, wdst, lane, *reinterpret_cast<const float2*>(&s.beta[16 * jb + 2 * t]),
                              *reinterpret_cast<const float2*>(&s.beta[16 * jb + 8 + 2 * t]));
                    if (!o) continue;
#pragma unroll
                    for (int ib = jb; ib < 4; ++ib) {
                        uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) {
                            uint32_t r[4];
                            ldm(r, pt + pl * (kYBlocks * 512) + tri(ib, jb) * 512);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NX, NX>(O[2 * ib], a, b0);
                        mma_planes<NX, NX, NX>(O[2 * ib + 1], a, b1);
                    }
                }
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    T* r0 = reinterpret_cast<T*>(stage + (8 * n + 2 * t) * kPitch);
                    T* r1 = reinterpret_cast<T*>(stage + (8 * n + 2 * t + 1) * kPitch);
                    r0[g] = from_f<T>(O[n][0]);
                    r1[g] = from_f<T>(O[n][1]);
                    r0[g + 8] = from_f<T>(O[n][2]);
                    r1[g + 8] = from_f<T>(O[n][3]);
                }
                __syncwarp();
            } else {
                bar_sync(1, 128);
            }
            const int col0 = c0 + 16 * w, width = min(16, p.e - col0);
            const bool whole = p.o.vec && width == 16;
            constexpr int kPieces = 16 * sizeof(T) / 16;  // 16-byte pieces of a row of 16 columns
            for (int i = lane; o && i < rows * kPieces; i += 32) {
                const int row = i / kPieces, piece = i % kPieces;
                T* dst = o + (n0 + row) * p.o.sn + col0;
                const bool live = s.any && s.live[row];
                const unsigned char* src = stage + row * kPitch + piece * 16;
                if (whole) {
                    reinterpret_cast<uint4*>(dst)[piece] =
                        live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
                } else {
                    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
                    for (int x = 0; x < kPer; ++x)
                        if (piece * kPer + x < width)
                            dst[piece * kPer + x] = live ? reinterpret_cast<const T*>(src)[x] : from_f<T>(0.f);
                }
            }
            __syncthreads();
        }
    } else {  // ---------------------------------------------------------- loads
        // the loads of a chunk are in flight for a whole iteration or two
        const int lt = tid - 128;
        const Gates* gates = p.gates + bh * p.nc;
        const bool outputs = p.o.p != nullptr;
        const int64_t kb = tensor_base(p.k, b, h), qb = tensor_base(p.q, b, h), vb = tensor_base(p.v, b, h);
        constexpr int kMat = NX * kYBlocks * 512;
        const unsigned char* Y = p.Y + bh * p.nc * kMat;
        const unsigned char* P = p.P + bh * p.nc * kMat;
        if (NIN == 1 && p.k.vec && p.q.vec && p.v.vec && p.d % 8 == 0 && p.e % 8 == 0) {
            // bf16: asynchronous copies, chunk c + 2 started while c is computed
            int any_next = gates[0].any;
            auto start = [&](int c) {
                if (c < p.nc) {
                    const int any = any_next;
                    any_next = c + 1 < p.nc ? gates[c + 1].any : 0;
                    auto& st = sm.st[c % NST];
                    async16<128>(reinterpret_cast<unsigned char*>(&st.s), reinterpret_cast<const unsigned char*>(gates + c), sizeof(Gates), lt);
                    if (any) {
                        const int n0 = c * kDeltaC;
                        async_tile<T, DP, 128>(st.k, p.k, kb, n0, 0, p.d, p.N, lt);
                        async_tile<T, kDeltaCols, 128>(st.v, p.v, vb, n0, c0, p.e, p.N, lt);
                        async16<128>(st.y, Y + (int64_t)c * kMat, kMat, lt);
                        if (outputs) {
                            async_tile<T, DP, 128>(st.q, p.q, qb, n0, 0, p.d, p.N, lt);
                            async16<128>(st.P, P + (int64_t)c * kMat, kMat, lt);
                        }
                    }
                }
                async_commit();
            };
            auto finish = [&](int c) {  // every copy but the last group's is there
                async_wait_but_one();
                if (c >= p.nc) return;
                bar_sync(3, 128);
                auto& st = sm.st[c % NST];
                if (st.s.any && !st.s.full) {
                    clear_dead<DP, 128>(st.k, st.s.live, lt);
                    clear_dead<DP, 128>(st.q, st.s.live, lt);
                    clear_dead<kDeltaCols, 128>(st.v, st.s.live, lt);
                }
            };
            start(0);
            start(1);
            finish(0);
            __syncthreads();
            for (int c = 0; c < p.nc; ++c) {
                start(c + 2);
                finish(c + 1);
                __syncthreads();
            }
            async_wait();
        } else {
            TileRegs<T, DP, 128> k, q;
            TileRegs<T, kDeltaCols, 128> v;
            ByteRegs<kMat, 128> y, P_;
            ByteRegs<sizeof(Gates), 128> s;
            int any = 0, any_next = gates[0].any;  // of the chunk in the registers, and of the one after it
            auto issue = [&](int c) {
                any = any_next;
                any_next = c + 1 < p.nc ? gates[c + 1].any : 0;
                if (c >= p.nc) return;
                s.issue(gates + c, lt);
                if (!any) return;
                const int n0 = c * kDeltaC;
                k.issue(p.k, kb, n0, 0, p.d, p.N, lt);
                v.issue(p.v, vb, n0, c0, p.e, p.N, lt);
                y.issue(Y + (int64_t)c * kMat, lt);
                if (outputs) {
                    q.issue(p.q, qb, n0, 0, p.d, p.N, lt);
                    P_.issue(P + (int64_t)c * kMat, lt);
                }
            };
            auto store = [&](int c) {
                if (c >= p.nc) return;
                auto& st = sm.st[c % NST];
                s.store(&st.s, lt);
                bar_sync(3, 128);
                if (!any) return;
                k.template store_planes<NIN>(st.k, st.s.live, lt);
                v.template store_planes<NIN>(st.v, st.s.live, lt);
                y.store(st.y, lt);
                if (outputs) {
                    q.template store_planes<NIN>(st.q, st.s.live, lt);
                    P_.store(st.P, lt);
                }
            };
            constexpr int kAhead = NST == 1 ? 0 : 1;
            issue(0);
            if (kAhead) {
                store(0);
                issue(1);
            }
            __syncthreads();
            for (int c = 0; c < p.nc; ++c) {
                store(c + kAhead);
                issue(c + kAhead + 1);
                if (NST == 1) __syncthreads();
                __syncthreads();
            }
        }
    }
}

template <typename T, int DP>
cudaError_t fwd_t(const DeltaParams& p, cudaStream_t st) {
    const int64_t bh = (int64_t)p.B * p.H, ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    const size_t prep = sizeof(PrepSmem<T, DP>), chain = sizeof(ChainSmem<T, DP>);
    static_assert(sizeof(ChainSmem<T, DP>) <= 227 * 1024, "shared memory");
    cudaError_t err = cudaFuncSetAttribute(delta_prep_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prep);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute(delta_chain_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)chain);
    if (err != cudaSuccess) return err;
    delta_prep_kernel<T, DP><<<(unsigned)(bh * p.nc), 128, prep, st>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    delta_chain_kernel<T, DP><<<(unsigned)(bh * ncb), 256, chain, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_delta_fwd(const DeltaParams& p, int dtype, cudaStream_t st) {
    if (p.d <= 64) {
        if (dtype == SUBQ_BF16) return fwd_t<__nv_bfloat16, 64>(p, st);
        if (dtype == SUBQ_FP16) return fwd_t<__half, 64>(p, st);
        return fwd_t<float, 64>(p, st);
    }
    if (dtype == SUBQ_BF16) return fwd_t<__nv_bfloat16, 128>(p, st);
    if (dtype == SUBQ_FP16) return fwd_t<__half, 128>(p, st);
    return fwd_t<float, 128>(p, st);
}

}  // namespace subq
