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
//   dlog gamma_t = sum over i >= t in the chunk of (q_i.dq_i - v_i.dv_i) + <G, S'>
// for all chunks at once (delta_grad_kernel). The last line is the scaling
// symmetry of the recurrence: multiplying S_t by e^{x_t} only moves factors
// between q_t, k_t and the gates, so g_i enters through q_i.dq_i and v_i.dv_i.
// <G, S'> = e^{g_C} <G, S0> + sum_j k_j.(D beta W G^T)_j.
#include "delta_common.cuh"
#include "delta_launch.h"
#include "scan_launch.h"

namespace subq {
namespace {

using namespace dl;

// ------------------------------------------------------------------ the walk back
template <typename T, int DP>
struct RevSmem {
    static constexpr int kIn = DeltaType<T>::kIn, kX = DeltaType<T>::kX;
    static constexpr int kStages = sizeof(T) == 4 && DP == 128 ? 1 : 2;
    struct Stage {
        alignas(128) unsigned char k[kIn * 64 * DP * 2];
        alignas(128) unsigned char q[kIn * 64 * DP * 2];
        alignas(128) unsigned char y[kX * kYBlocks * 512];
        alignas(128) unsigned char g[kIn * 64 * kDeltaCols * 2];  // dO
        Gates s;
    } st[kStages];
    alignas(128) unsigned char P[kX * kYBlocks * 512];
    alignas(16) float e1[2][8 * 128];       // (P^T dO)^T accumulators per warp of 16 columns
    alignas(16) float e2[2][DP / 8 * 128];  // (scale (e^g Q)^T dO)^T
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, 1) delta_rev_kernel(const DeltaParams p) {
    constexpr int NIN = DeltaType<T>::kIn, NX = DeltaType<T>::kX, kTile = 64 * DP * 2, kGTile = 64 * kDeltaCols * 2;
    constexpr int NST = RevSmem<T, DP>::kStages;
    extern __shared__ __align__(128) unsigned char raw[];
    RevSmem<T, DP>& sm = *reinterpret_cast<RevSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    const int64_t bh = blockIdx.x / ncb;
    const int cb = blockIdx.x % ncb, b = (int)(bh / p.H), h = (int)(bh % p.H), c0 = cb * kDeltaCols;
    const int g = lane >> 2, t = lane & 3;

    auto load_stage = [&](int c) {
        auto& st = sm.st[c % NST];
        const int lt = tid - 128, n0 = c * kDeltaC;
        if (warp == 4) load_gates(st.s, p, b, h, n0, lane);
        bar_sync(3, 128);
        if (!st.s.any) return;
        load_planes<T, DP, NIN, 128>(st.k, p.k, tensor_base(p.k, b, h), n0, 0, p.d, st.s.live, lt);
        load_planes<T, DP, NIN, 128>(st.q, p.q, tensor_base(p.q, b, h), n0, 0, p.d, st.s.live, lt);
        load_planes<T, kDeltaCols, NIN, 128>(st.g, p.g, tensor_base(p.g, b, h), n0, c0, p.e, st.s.live, lt);
        copy16<128>(st.y, p.Y + (bh * p.nc + c) * (NX * kYBlocks * 512), NX * kYBlocks * 512, lt);
    };

    if (warp < 2) {  // ---------------------------------------------------- chain
        float S[DP / 8][4];  // G^T: 16 value columns x d
        const int col0 = c0 + 16 * warp;
        const float* G_in = p.dS_out ? p.dS_out + bh * p.d * p.e : nullptr;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 8 * n + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
                S[n][i] = (G_in && d < p.d && col < p.e) ? G_in[(int64_t)d * p.e + col] : 0.f;
            }
        const int64_t cw = 2 * cb + warp, ncw = 2 * ncb;
        bool pending = false;  // e2 of the chunk before has to be added
        auto add_e2 = [&]() {
            const float4* e2 = reinterpret_cast<const float4*>(sm.e2[warp]);
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
                const float4 x = e2[n * 32 + lane];
                S[n][0] += x.x; S[n][1] += x.y; S[n][2] += x.z; S[n][3] += x.w;
            }
        };
        __syncthreads();
        for (int c = p.nc - 1; c >= 0; --c) {
            if (NST == 1) __syncthreads();
            auto& st = sm.st[c % NST];
            const Gates& s = st.s;
            if (pending) add_e2();
            pending = s.any;
            if (s.any) {
                const uint32_t kt = smem_addr(st.k);
                unsigned char* gdst = p.dS + ((bh * p.nc + c) * ncw + cw) * (DP / 16 * NX * 512) + lane * 4;
                float X[8][4];
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) X[n][i] = 0.f;
                const float2 one = make_float2(1.f, 1.f);
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {  // (K G)^T
                    uint32_t a[NX][4];
                    to_a<NX>(S[2 * kk], S[2 * kk + 1], one, one, a);
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl)
#pragma unroll
                        for (int m = 0; m < 4; ++m)
                            *reinterpret_cast<uint32_t*>(gdst + (kk * NX + pl) * 512 + m * 128) = a[pl][m];
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
                bar_sync(1, 128);  // e1 is there, and e2 of the chunk before has been read
                const float4* e1 = reinterpret_cast<const float4*>(sm.e1[warp]);
#pragma unroll
                for (int n = 0; n < 8; ++n) {  // dU^T
                    const float4 x = e1[n * 32 + lane];
                    const float2 kd = *reinterpret_cast<const float2*>(&s.kd[8 * n + 2 * t]);
                    X[n][0] = fmaf(kd.x, X[n][0], x.x);
                    X[n][1] = fmaf(kd.y, X[n][1], x.y);
                    X[n][2] = fmaf(kd.x, X[n][2], x.z);
                    X[n][3] = fmaf(kd.y, X[n][3], x.w);
                }
                uint32_t ra[4][NX][4];
#pragma unroll
                for (int ib = 0; ib < 4; ++ib) {
                    const float2 b0 = *reinterpret_cast<const float2*>(&s.beta[16 * ib + 2 * t]);
                    const float2 b1 = *reinterpret_cast<const float2*>(&s.beta[16 * ib + 8 + 2 * t]);
                    to_a<NX>(X[2 * ib], X[2 * ib + 1], make_float2(-b0.x, -b0.y), make_float2(-b1.x, -b1.y), ra[ib]);
                }
                // Z^T = dU^T - (beta dU)^T Y
                const uint32_t yt = smem_addr(st.y) + lane * 16;
#pragma unroll
                for (int jb = 0; jb < 4; ++jb)
#pragma unroll
                    for (int ib = jb; ib < 4; ++ib) {
                        uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) {
                            uint32_t r[4];
                            ldm_t(r, yt + pl * (kYBlocks * 512) + tri(ib, jb) * 512);
                            b0[pl][0] = r[0]; b0[pl][1] = r[2]; b1[pl][0] = r[1]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NX, NX>(X[2 * jb], ra[ib], b0);
                        mma_planes<NX, NX, NX>(X[2 * jb + 1], ra[ib], b1);
                    }
                unsigned char* zdst = p.Z + ((bh * p.nc + c) * ncw + cw) * (4 * NX * 512) + lane * 4;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[n][i] *= s.eC;
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    uint32_t a[NX][4];
                    to_a<NX>(X[2 * jb], X[2 * jb + 1], one, one, a);
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl)
#pragma unroll
                        for (int m = 0; m < 4; ++m)
                            *reinterpret_cast<uint32_t*>(zdst + (jb * NX + pl) * 512 + m * 128) = a[pl][m];
                    float2 f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = 16 * jb + 8 * i + 2 * t;
                        f[i] = make_float2(-s.beta[j] * s.eg[j], -s.beta[j + 1] * s.eg[j + 1]);
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
            }
            __syncthreads();
        }
        if (pending) add_e2();
        if (p.dS_in) {
            float* G_out = p.dS_in + bh * p.d * p.e;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 8 * n + 2 * t + (i & 1), col = col0 + g + 8 * (i >> 1);
                    if (d < p.d && col < p.e) G_out[(int64_t)d * p.e + col] = S[n][i];
                }
        }
    } else if (warp < 4) {  // ------------------------------- P^T dO and (e^g Q)^T dO
        const int w = warp - 2;
        __syncthreads();
        for (int c = p.nc - 1; c >= 0; --c) {
            if (NST == 1) __syncthreads();
            auto& st = sm.st[c % NST];
            const Gates& s = st.s;
            if (s.any) {
                const uint32_t kt = smem_addr(st.k), qt = smem_addr(st.q), gt = smem_addr(st.g);
                score_rows<DP, NIN, NX>(sm.P, qt, kt, s, p.scale, false, w ? 1 : 0, lane);
                score_rows<DP, NIN, NX>(sm.P, qt, kt, s, p.scale, false, w ? 2 : 3, lane);
                bar_sync(2, 64);
                uint32_t da[4][NIN][4];  // dO^T: 16 value columns x 64 tokens
#pragma unroll
                for (int ib = 0; ib < 4; ++ib)
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) a_cols<kDeltaCols>(da[ib][pl], gt + pl * kGTile, 16 * ib, w, lane);
                const uint32_t pt = smem_addr(sm.P) + lane * 16;
                float4* e1 = reinterpret_cast<float4*>(sm.e1[w]);
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ib = jb; ib < 4; ++ib) {
                        uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) {
                            uint32_t r[4];
                            ldm_t(r, pt + pl * (kYBlocks * 512) + tri(ib, jb) * 512);
                            b0[pl][0] = r[0]; b0[pl][1] = r[2]; b1[pl][0] = r[1]; b1[pl][1] = r[3];
                        }
                        mma_planes<NIN, NX, NX>(a0, da[ib], b0);
                        mma_planes<NIN, NX, NX>(a1, da[ib], b1);
                    }
                    e1[(2 * jb) * 32 + lane] = make_float4(a0[0], a0[1], a0[2], a0[3]);
                    e1[(2 * jb + 1) * 32 + lane] = make_float4(a1[0], a1[1], a1[2], a1[3]);
                }
                bar_sync(1, 128);
                float E[DP / 8][4];
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) E[n][i] = 0.f;
#pragma unroll
                for (int ib = 0; ib < 4; ++ib) {
                    uint32_t a[NX][4];
#pragma unroll
                    for (int m = 0; m < 4; ++m) {  // scale e^g dO, tokens 16 ib + 8 (m / 2) + 2 t, + 1
                        float x = 0.f, y = 0.f;
#pragma unroll
                        for (int pl = 0; pl < NIN; ++pl) {
                            const float2 u = unpack_bf16(da[ib][pl][m]);
                            x += u.x;
                            y += u.y;
                        }
                        const int i = 16 * ib + 8 * (m >> 1) + 2 * t;
                        uint32_t r[NX];
                        split2<NX>(x * p.scale * s.eg[i], y * p.scale * s.eg[i + 1], r);
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) a[pl][m] = r[pl];
                    }
#pragma unroll
                    for (int np = 0; np < DP / 16; ++np) {
                        uint32_t b0[NIN][2], b1[NIN][2];
#pragma unroll
                        for (int pl = 0; pl < NIN; ++pl) {
                            uint32_t r[4];
                            b_cols<DP>(r, qt + pl * kTile, 16 * ib, np, lane);
                            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                        }
                        mma_planes<NX, NIN, NX>(E[2 * np], a, b0);
                        mma_planes<NX, NIN, NX>(E[2 * np + 1], a, b1);
                    }
                }
                float4* e2 = reinterpret_cast<float4*>(sm.e2[w]);
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) e2[n * 32 + lane] = make_float4(E[n][0], E[n][1], E[n][2], E[n][3]);
            }
            __syncthreads();
        }
    } else {  // ---------------------------------------------------------- loads
        if (NST == 2) load_stage(p.nc - 1);
        __syncthreads();
        for (int c = p.nc - 1; c >= 0; --c) {
            if (NST == 1) {
                load_stage(c);
                __syncthreads();
            } else if (c > 0) {
                load_stage(c - 1);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ the gradients
template <typename T, int DP>
struct GradSmem {
    static constexpr int kIn = DeltaType<T>::kIn, kX = DeltaType<T>::kX;
    Gates s;
    float qdq[2][kDeltaC], vdv[kDeltaC], wz[kDeltaC], kdk[2][kDeltaC];
    float gs[8];
    alignas(128) unsigned char k[kIn * 64 * DP * 2];
    alignas(128) unsigned char q[kIn * 64 * DP * 2];
    union {
        struct {  // one block of 32 value columns
            alignas(128) unsigned char S0[2 * DP / 16 * kX * 512];
            alignas(128) unsigned char G[2 * DP / 16 * kX * 512];
            alignas(128) unsigned char W[2 * 4 * kX * 512];
            alignas(128) unsigned char Z[2 * 4 * kX * 512];
            alignas(128) unsigned char dO[kIn * 64 * kDeltaCols * 2];
        } in;
        struct {
            alignas(128) unsigned char d1[kX * kYBlocks * 512];
            alignas(128) unsigned char d2[kX * kYBlocks * 512];
        } sc;
    } u;
};

__device__ __forceinline__ float bf16_at(const unsigned char* p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
}

template <typename T, int DP>
__global__ void __launch_bounds__(256, 1) delta_grad_kernel(const DeltaParams p) {
    constexpr int NIN = DeltaType<T>::kIn, NX = DeltaType<T>::kX, kTile = 64 * DP * 2, kGTile = 64 * kDeltaCols * 2;
    constexpr int NB = DP / 16;  // 8-column blocks of a warp's half of d
    extern __shared__ __align__(128) unsigned char raw[];
    GradSmem<T, DP>& sm = *reinterpret_cast<GradSmem<T, DP>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int rb = warp & 3, hf = warp >> 2;  // 16 tokens, half of d
    const int64_t chunk = blockIdx.x, bh = chunk / p.nc;
    const int c = (int)(chunk % p.nc), b = (int)(bh / p.H), h = (int)(bh % p.H), n0 = c * kDeltaC;
    const int rows = min(kDeltaC, p.N - n0);
    const int ncb = (p.e + kDeltaCols - 1) / kDeltaCols;
    if (warp == 0) load_gates(sm.s, p, b, h, n0, lane);
    if (tid < kDeltaC) sm.vdv[tid] = sm.wz[tid] = 0.f;
    __syncthreads();
    const Gates& s = sm.s;

    // where the rows of this state head's gradients go
    auto grad_row = [&](const DeltaTensor& x, float* x32, int width, int n, T*& row, float*& row32) {
        row = nullptr;
        row32 = nullptr;
        if (x32) row32 = x32 + ((int64_t)bh * p.N + n) * width;
        else row = static_cast<T*>(x.p) + tensor_base(x, b, h) + n * x.sn;
    };

    float dq[NB][4], dk1[NB][4], dk2[NB][4], D[8][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) dq[n][i] = dk1[n][i] = dk2[n][i] = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) D[n][i] = 0.f;  // dO W^T (hf = 0) or Z W^T (hf = 1), rows 16 rb ..
    float gs = 0.f;

    if (s.any) {
        load_planes<T, DP, NIN, 256>(sm.k, p.k, tensor_base(p.k, b, h), n0, 0, p.d, s.live, tid);
        load_planes<T, DP, NIN, 256>(sm.q, p.q, tensor_base(p.q, b, h), n0, 0, p.d, s.live, tid);
    }
    for (int eb = 0; eb < ncb; ++eb) {
        if (s.any) {
            const int64_t at = chunk * 2 * ncb + 2 * eb;
            copy16<256>(sm.u.in.S0, p.S0 + at * (DP / 16 * NX * 512), 2 * DP / 16 * NX * 512, tid);
            copy16<256>(sm.u.in.G, p.dS + at * (DP / 16 * NX * 512), 2 * DP / 16 * NX * 512, tid);
            copy16<256>(sm.u.in.W, p.W + at * (4 * NX * 512), 2 * 4 * NX * 512, tid);
            copy16<256>(sm.u.in.Z, p.Z + at * (4 * NX * 512), 2 * 4 * NX * 512, tid);
            load_planes<T, kDeltaCols, NIN, 256>(sm.u.in.dO, p.g, tensor_base(p.g, b, h), n0, eb * kDeltaCols, p.e, s.live, tid);
            __syncthreads();
            const uint32_t S0 = smem_addr(sm.u.in.S0) + lane * 16, G = smem_addr(sm.u.in.G) + lane * 16;
            const uint32_t W = smem_addr(sm.u.in.W) + lane * 16, Z = smem_addr(sm.u.in.Z) + lane * 16;
            const uint32_t dO = smem_addr(sm.u.in.dO);
#pragma unroll
            for (int cw = 0; cw < 2; ++cw) {  // 16 value columns: one k step
                uint32_t ao[NIN][4], aw[NX][4], az[NX][4];
#pragma unroll
                for (int pl = 0; pl < NIN; ++pl) a_rows<kDeltaCols>(ao[pl], dO + pl * kGTile, 16 * rb, cw, lane);
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    uint32_t r[4];
                    ldm_t(r, W + ((cw * 4 + rb) * NX + pl) * 512);
                    aw[pl][0] = r[0]; aw[pl][1] = r[2]; aw[pl][2] = r[1]; aw[pl][3] = r[3];
                    ldm_t(r, Z + ((cw * 4 + rb) * NX + pl) * 512);
                    az[pl][0] = r[0]; az[pl][1] = r[2]; az[pl][2] = r[1]; az[pl][3] = r[3];
                }
#pragma unroll
                for (int n = 0; n < NB / 2; ++n) {
                    const int kk = hf * (NB / 2) + n;
                    uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl) {
                        uint32_t r[4];
                        ldm_t(r, S0 + ((cw * (DP / 16) + kk) * NX + pl) * 512);
                        b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                    }
                    mma_planes<NIN, NX, NX>(dq[2 * n], ao, b0);
                    mma_planes<NIN, NX, NX>(dq[2 * n + 1], ao, b1);
                    mma_planes<NX, NX, NX>(dk2[2 * n], az, b0);
                    mma_planes<NX, NX, NX>(dk2[2 * n + 1], az, b1);
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl) {
                        uint32_t r[4];
                        ldm_t(r, G + ((cw * (DP / 16) + kk) * NX + pl) * 512);
                        b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                    }
                    mma_planes<NX, NX, NX>(dk1[2 * n], aw, b0);
                    mma_planes<NX, NX, NX>(dk1[2 * n + 1], aw, b1);
                }
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    if (jb > rb) continue;
                    uint32_t b0[NX][2], b1[NX][2];
#pragma unroll
                    for (int pl = 0; pl < NX; ++pl) {
                        uint32_t r[4];
                        ldm_t(r, W + ((cw * 4 + jb) * NX + pl) * 512);
                        b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
                    }
                    if (hf == 0) {
                        mma_planes<NIN, NX, NX>(D[2 * jb], ao, b0);
                        mma_planes<NIN, NX, NX>(D[2 * jb + 1], ao, b1);
                    } else {
                        mma_planes<NX, NX, NX>(D[2 * jb], az, b0);
                        mma_planes<NX, NX, NX>(D[2 * jb + 1], az, b1);
                    }
                }
            }
        }
        {  // dv = beta Z, and the row sums W.Z and v.dv: a token and 8 value columns per thread
            const int tok = tid & 63, grp = tid >> 6, cw = grp >> 1, col = eb * kDeltaCols + grp * 8;
            float wz = 0.f, vdv = 0.f;
            if (tok < rows && col < p.e) {
                const int n = n0 + tok;
                const bool on = s.any && s.live[tok];
                T* row;
                float* row32;
                grad_row(p.dv, p.dv32, p.e, n, row, row32);
                const T* v = static_cast<const T*>(p.v.p) + tensor_base(p.v, b, h) + n * p.v.sn;
                T ov[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float z = 0.f, w = 0.f;
                    if (on) {
                        // element (value column 8 (grp % 2) + i, token): matrix [token half][column half], row i
                        const int off = (((tok >> 3) & 1) * 2 + (grp & 1)) * 128 + i * 16 + (tok & 7) * 2;
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl) {
                            const int tile = ((cw * 4 + (tok >> 4)) * NX + pl) * 512;
                            z += bf16_at(sm.u.in.Z + tile + off);
                            w += bf16_at(sm.u.in.W + tile + off);
                        }
                    }
                    wz = fmaf(w, z, wz);
                    z *= s.beta[tok];
                    if (on && col + i < p.e) vdv = fmaf(z, to_f<T>(v[col + i]), vdv);
                    ov[i] = from_f<T>(z);
                    if (row32 && col + i < p.e) row32[col + i] = z;
                }
                if (row) {
                    if (p.dv.vec && col + 8 <= p.e) {
#pragma unroll
                        for (int x = 0; x < (int)sizeof(T) / 2; ++x)
                            reinterpret_cast<uint4*>(row + col)[x] = reinterpret_cast<const uint4*>(ov)[x];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (col + i < p.e) row[col + i] = ov[i];
                    }
                }
            }
            // fixed order: the four groups add one after the other
            for (int x = 0; x < 4; ++x) {
                if (grp == x) {
                    sm.wz[tok] += wz;
                    sm.vdv[tok] += vdv;
                }
                __syncthreads();
            }
        }
        if (s.any) {  // <G, S0>
            for (int i = tid; i < 2 * DP / 16 * 128; i += 256) {
                const int tile = i >> 7, off = (i & 127) * 4;
                float2 x = make_float2(0.f, 0.f), y = x;
#pragma unroll
                for (int pl = 0; pl < NX; ++pl) {
                    const float2 u0 = unpack_bf16(*reinterpret_cast<const uint32_t*>(sm.u.in.S0 + (tile * NX + pl) * 512 + off));
                    const float2 u1 = unpack_bf16(*reinterpret_cast<const uint32_t*>(sm.u.in.G + (tile * NX + pl) * 512 + off));
                    x.x += u0.x; x.y += u0.y;
                    y.x += u1.x; y.y += u1.y;
                }
                gs = fmaf(x.x, y.x, gs);
                gs = fmaf(x.y, y.y, gs);
            }
            __syncthreads();
        }
    }

    if (s.any) {
        {  // D1 or D2 as planes
            unsigned char* dst = hf ? sm.u.sc.d2 : sm.u.sc.d1;
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {
                if (jb > rb) continue;
#pragma unroll
                for (int jh = 0; jh < 2; ++jh)
#pragma unroll
                    for (int ih = 0; ih < 2; ++ih) {
                        const int i = 16 * rb + 8 * ih + g, j = 16 * jb + 8 * jh + 2 * t;
                        const float fi = hf ? -s.beta[i] : p.scale;
                        float x = 0.f, y = 0.f;
                        if (j < i || (j == i && !hf)) x = fi * s.beta[j] * gamma_ij(s, i, j) * D[2 * jb + jh][2 * ih];
                        if (j + 1 < i || (j + 1 == i && !hf))
                            y = fi * s.beta[j + 1] * gamma_ij(s, i, j + 1) * D[2 * jb + jh][2 * ih + 1];
                        uint32_t r[NX];
                        split2<NX>(x, y, r);
#pragma unroll
                        for (int pl = 0; pl < NX; ++pl)
                            *reinterpret_cast<uint32_t*>(dst + (pl * kYBlocks + tri(rb, jb)) * 512 + (ih * 2 + jh) * 128 + lane * 4) = r[pl];
                    }
            }
        }
        // row factors of the products with the states; k.dk1 before anything is added to it
        {
            float kd[2] = {0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = 16 * rb + 8 * x + g;
                const float fq = p.scale * s.eg[i], f1 = s.kd[i] * s.beta[i], f2 = -s.eg[i] * s.beta[i];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const int piece = hf * NB + n;
                    float2 kv = make_float2(0.f, 0.f);
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) {
                        const float2 u = unpack_bf16(*reinterpret_cast<const uint32_t*>(sm.k + pl * kTile + tile_off<DP>(i, piece) + 4 * t));
                        kv.x += u.x;
                        kv.y += u.y;
                    }
                    const float a = f1 * dk1[n][2 * x], d = f1 * dk1[n][2 * x + 1];
                    kd[x] = fmaf(a, kv.x, kd[x]);
                    kd[x] = fmaf(d, kv.y, kd[x]);
                    dk1[n][2 * x] = fmaf(f2, dk2[n][2 * x], a);
                    dk1[n][2 * x + 1] = fmaf(f2, dk2[n][2 * x + 1], d);
                    dq[n][2 * x] *= fq;
                    dq[n][2 * x + 1] *= fq;
                }
                kd[x] += __shfl_xor_sync(0xffffffffu, kd[x], 1);
                kd[x] += __shfl_xor_sync(0xffffffffu, kd[x], 2);
                if (t == 0) sm.kdk[hf][i] = kd[x];
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
                    mma_planes<NX, NIN, NX>(dq[2 * n], a1, k0);
                    mma_planes<NX, NIN, NX>(dq[2 * n + 1], a1, k1);
                    mma_planes<NX, NIN, NX>(dk1[2 * n], a2, k0);
                    mma_planes<NX, NIN, NX>(dk1[2 * n + 1], a2, k1);
                }
                if (ob >= rb) {
                    mma_planes<NX, NIN, NX>(dk1[2 * n], a1t, q0);
                    mma_planes<NX, NIN, NX>(dk1[2 * n + 1], a1t, q1);
                    mma_planes<NX, NIN, NX>(dk1[2 * n], a2t, k0);
                    mma_planes<NX, NIN, NX>(dk1[2 * n + 1], a2t, k1);
                }
            }
        }
        {  // q.dq
            float qd[2] = {0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = 16 * rb + 8 * x + g;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int pl = 0; pl < NIN; ++pl) {
                        const float2 u = unpack_bf16(
                            *reinterpret_cast<const uint32_t*>(sm.q + pl * kTile + tile_off<DP>(i, hf * NB + n) + 4 * t));
                        qd[x] = fmaf(u.x, dq[n][2 * x], qd[x]);
                        qd[x] = fmaf(u.y, dq[n][2 * x + 1], qd[x]);
                    }
                qd[x] += __shfl_xor_sync(0xffffffffu, qd[x], 1);
                qd[x] += __shfl_xor_sync(0xffffffffu, qd[x], 2);
                if (t == 0) sm.qdq[hf][i] = qd[x];
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) gs += __shfl_xor_sync(0xffffffffu, gs, o);
        if (lane == 0) sm.gs[warp] = gs;
    }
    // dq and dk rows: quads hold neighbouring columns
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int i = 16 * rb + 8 * x + g;
        if (i >= rows) continue;
        T *rq, *rk;
        float *rq32, *rk32;
        grad_row(p.dq, p.dq32, p.d, n0 + i, rq, rq32);
        grad_row(p.dk, p.dk32, p.d, n0 + i, rk, rk32);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int col = (hf * NB + n) * 8 + 2 * t;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (col + y >= p.d) continue;
                if (rq32) rq32[col + y] = dq[n][2 * x + y];
                else rq[col + y] = from_f<T>(dq[n][2 * x + y]);
                if (rk32) rk32[col + y] = dk1[n][2 * x + y];
                else rk[col + y] = from_f<T>(dk1[n][2 * x + y]);
            }
        }
    }
    __syncthreads();
    if (warp == 0) {
        // suffix sums over the chunk (two tokens per lane) on top of <G, S'>
        const int i0 = 2 * lane, i1 = i0 + 1;
        float x0 = 0.f, x1 = 0.f, k01 = 0.f, end = 0.f;
        if (s.any) {
            x0 = sm.qdq[0][i0] + sm.qdq[1][i0] - sm.vdv[i0];
            x1 = sm.qdq[0][i1] + sm.qdq[1][i1] - sm.vdv[i1];
            k01 = sm.kdk[0][i0] + sm.kdk[1][i0] + sm.kdk[0][i1] + sm.kdk[1][i1];
            for (int w = 0; w < 8; ++w) end += sm.gs[w];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) k01 += __shfl_xor_sync(0xffffffffu, k01, o);
        end = s.eC * end + k01;
        float run = x0 + x1;  // suffix sum over lanes >= this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float down = __shfl_down_sync(0xffffffffu, run, o);
            if (lane + o < 32) run += down;
        }
        const int64_t at = bh * p.N + n0;
        if (i0 < rows) {
            p.dbeta[at + i0] = s.any && s.live[i0] ? sm.wz[i0] : 0.f;
            if (p.dlg) p.dlg[at + i0] = s.any && s.live[i0] ? run + end : 0.f;
        }
        if (i1 < rows) {
            p.dbeta[at + i1] = s.any && s.live[i1] ? sm.wz[i1] : 0.f;
            if (p.dlg) p.dlg[at + i1] = s.any && s.live[i1] ? run - x0 + end : 0.f;
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
    cudaError_t err = cudaFuncSetAttribute(delta_rev_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rev);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute(delta_grad_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)grad);
    if (err != cudaSuccess) return err;
    delta_rev_kernel<T, DP><<<(unsigned)(bh * ncb), 256, rev, st>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    delta_grad_kernel<T, DP><<<(unsigned)(bh * p.nc), 256, grad, st>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    *launches = 2;
    if ((err = group_sum<T>(p.dq32, p.dq, p, p.d, st, launches)) != cudaSuccess) return err;
    if ((err = group_sum<T>(p.dk32, p.dk, p, p.d, st, launches)) != cudaSuccess) return err;
    return group_sum<T>(p.dv32, p.dv, p, p.e, st, launches);
}

}  // namespace

cudaError_t launch_delta_bwd(const DeltaParams& p, int dtype, cudaStream_t st, int* launches) {
    if (p.d <= 64) {
        if (dtype == SUBQ_BF16) return bwd_t<__nv_bfloat16, 64>(p, st, launches);
        if (dtype == SUBQ_FP16) return bwd_t<__half, 64>(p, st, launches);
        return bwd_t<float, 64>(p, st, launches);
    }
    if (dtype == SUBQ_BF16) return bwd_t<__nv_bfloat16, 128>(p, st, launches);
    if (dtype == SUBQ_FP16) return bwd_t<__half, 128>(p, st, launches);
    return bwd_t<float, 128>(p, st, launches);
}

}  // namespace subq
