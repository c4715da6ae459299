// Shared pieces of the gated delta rule kernels (delta_step.cu, delta_fwd.cuh,
// delta_bwd.cuh). Per (batch, head) sequence with live tokens t:
//   S_t = gamma_t S_{t-1} + beta_t k_t w_t^T,   w_t = v_t - gamma_t S_{t-1}^T k_t,
//   o_t = scale S_t^T q_t;   a masked token leaves S as it is and has o = 0.
//
// Chunk form (C = 64 tokens from the state S0; g = running sum of log gamma in
// the chunk, G_ij = exp(g_i - g_j) for i >= j, A_ij = G_ij k_i.k_j for i > j):
//   R = V - e^g (K S0),   W = R - Y (beta R),   Y = (I + A beta)^-1 A
//   O = scale (e^g (Q S0) + (G o Q K^T) (beta W))
//   S' = e^{g_C} S0 + K^T (e^{g_C - g} beta W)
// Y is strictly lower triangular and depends on k and the gates alone, so it is
// formed for all chunks at once; the walk over the chunks is two products deep.
//
// Precision: operands go through the bf16 tensor-core instruction as sums of
// bf16 planes (a float is hi + mid + lo to 2^-25, relative), products accumulate
// in float32. Inputs are held exactly (bf16: 1 plane, fp16: 2, fp32: 3); what is
// computed in between (states, W, Y, scores) is held in three planes for every
// type, and plane products whose planes' indices sum to 3 or more are below that
// precision and left out. (Two planes for 16-bit inputs would take 0.7 of the
// time, but turn one rounding of a bf16 output in a thousand and leave float32
// results 3e-6 to 8e-6 off instead of 3e-7 to 6e-7.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.hpp"
#include "scan_common.cuh"

namespace subq {

struct DeltaTensor {
    void* p;
    int64_t sb, sh, sn;
    int group;  // heads of the state per head of this tensor
    int vec;    // rows start on 16-byte boundaries and hold a multiple of 8 elements
};

struct DeltaGate {
    const float* p;  // null: the neutral value
    int64_t sb, sh, sn;
};

struct DeltaParams {
    int B, H, N, d, e;
    int nc;  // chunks of 64 tokens
    float scale;
    DeltaGate beta, lg;
    const uint8_t* mask;
    int64_t mask_sb;
    DeltaTensor q, k, v, o;
    const float* S_in;  // [B, H, d, e]
    float* S_out;
    struct DeltaGates* gates;  // [B * H][nc]
    unsigned char* Y;   // Y^T: [B * H][nc][NX][10 blocks of 512 bytes]
    unsigned char* P;   // scale G o (Q K^T), likewise
    unsigned char* S0;  // [B * H][nc][ep / 16][dp / 16][NX][512], or null (not stored)
    unsigned char* W;   // [B * H][nc][ep / 16][4][NX][512], or null
    // segments of a sequence walked side by side (few sequences): 1, or more than 1 with `seg_S` and `seg_M`
    int nseg, seg_chunks;
    float* seg_S;  // [B * H][nseg - 1][d, e]: state after a segment
    float* seg_M;  // [B * H][nseg - 1][dp, dp] (d padded): what a segment does to the state before it, transposed
    float* seg_in;  // [B * H][d, e]: copy of S_in where S_out is S_in (one CTA reads it, another writes it), else null
    // backward
    DeltaTensor g, dq, dk, dv;
    unsigned char* dS;  // gradient of the state after each chunk, like S0
    unsigned char* Z;   // like W
    float* dq32;        // [B, H, N, d] per state head when q is shared by a group, else null
    float* dk32;
    float* dv32;        // [B, H, N, e]
    const float* dS_out;  // gradient of the final state, or null
    float* dS_in;         // gradient of the initial state, or null
    float* dbeta;         // [B, H, N]
    float* dlg;           // [B, H, N] or null
};

constexpr int kDeltaC = 64;      // tokens per chunk
constexpr int kDeltaCols = 32;   // value columns per CTA of the chunk walks
constexpr int kYBlocks = 10;     // 16 x 16 blocks of the lower triangle of a 64 x 64 matrix
constexpr float kMinLogGamma = -120.f;  // exp() of anything lower is 0 in float32 as well

// Gates of one chunk, formed once (delta_prep_kernel) and read by every kernel.
struct alignas(16) DeltaGates {
    float gh[kDeltaC], gl[kDeltaC];  // running sum of log2 gamma: g / ln 2 = gh + gl
    float beta[kDeltaC];             // 0 on masked tokens
    float eg[kDeltaC];               // e^g
    float kd[kDeltaC];               // e^{g_C - g}
    int live[kDeltaC];
    float eC, dC;                    // e^{g_C}, e^{g_C} - 1
    int any, full;                   // a live token in the chunk; all 64 live
};
static_assert(sizeof(DeltaGates) % 16 == 0 && sizeof(DeltaGates) <= 128 * 16, "one 16-byte piece per loading thread");

constexpr int kDeltaPlanes = 3;  // of what is computed in between
template <typename T> constexpr int kDeltaIn = sizeof(T) == 4 ? 3 : 2;  // of inputs
template <> constexpr int kDeltaIn<__nv_bfloat16> = 1;

namespace dl {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices of 16-bit elements; lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// (x, y) as NP pairs of bf16 whose sums are x and y to NP * 8 bits. An infinity
// or NaN stays what it is in plane 0 and leaves NaN in the others.
template <int NP>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&r)[NP]) {
    r[0] = pack_bf16(x, y);
#pragma unroll
    for (int i = 1; i < NP; ++i) {
        const float2 h = unpack_bf16(r[i - 1]);
        x -= h.x;
        y -= h.y;
        r[i] = pack_bf16(x, y);
    }
}

// c[n] += A B[n], plane pair by plane pair over all n: each accumulator is used again only after the others, which
// hides the instruction's latency (22 cycles against 8 of issue: four accumulators at least).
// The tensor cores cut a sum off where float32 addition rounds it, so every instruction on an accumulator loses up to
// 2^-23 of it, always towards zero. The small products (planes' indices not both 0) are therefore summed by themselves and
// added once: outputs of float32 inputs are then off by 4.4e-7 (2.6e-6 with one sum), for 5 % of the time of a training step.
template <int N, int NA, int NB, int NX>
__device__ __forceinline__ void mma_set(float (&c)[N][4], const uint32_t (&a)[NA][4], const uint32_t (&b)[N][NB][2]) {
    constexpr bool kSmall = NA * NB > 1;
    float small[N][4];
    if constexpr (kSmall) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) small[n][i] = 0.f;
    }
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j < NX)
#pragma unroll
                for (int n = 0; n < N; ++n) mma(i + j > 0 ? small[n] : c[n], a[i], b[n][j][0], b[n][j][1]);
    if constexpr (kSmall) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[n][i] += small[n][i];
    }
}
template <int NA, int NB, int NX>
__device__ __forceinline__ void mma_pair(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b0)[NB][2],
                                         const uint32_t (&b1)[NB][2]) {
    constexpr bool kSmall = NA * NB > 1;
    float small[2][4];
    if constexpr (kSmall) {
#pragma unroll
        for (int i = 0; i < 4; ++i) small[0][i] = small[1][i] = 0.f;
    }
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j < NX) {
                mma(i + j > 0 ? small[0] : c0, a[i], b0[j][0], b0[j][1]);
                mma(i + j > 0 ? small[1] : c1, a[i], b1[j][0], b1[j][1]);
            }
    if constexpr (kSmall) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c0[i] += small[0][i];
            c1[i] += small[1][i];
        }
    }
}

// Accumulators of two neighbouring 8-column blocks (16 rows x 16 columns) as the
// A operand of the next product, times per-column factors f0 (columns 2t, 2t + 1
// of the first block) and f1 (of the second).
template <int NX>
__device__ __forceinline__ void to_a(const float (&c0)[4], const float (&c1)[4], float2 f0, float2 f1, uint32_t (&a)[NX][4]) {
    uint32_t r[NX];
    split2<NX>(c0[0] * f0.x, c0[1] * f0.y, r);
#pragma unroll
    for (int i = 0; i < NX; ++i) a[i][0] = r[i];
    split2<NX>(c0[2] * f0.x, c0[3] * f0.y, r);
#pragma unroll
    for (int i = 0; i < NX; ++i) a[i][1] = r[i];
    split2<NX>(c1[0] * f1.x, c1[1] * f1.y, r);
#pragma unroll
    for (int i = 0; i < NX; ++i) a[i][2] = r[i];
    split2<NX>(c1[2] * f1.x, c1[3] * f1.y, r);
#pragma unroll
    for (int i = 0; i < NX; ++i) a[i][3] = r[i];
}

// ---- shared-memory tiles
// Row-major [64][W] bf16 planes in 16-byte pieces; the piece index is XORed so
// that 8 consecutive rows of one piece column fall into 8 different bank groups
// (ldmatrix and the 16-byte stores are then free of conflicts).
template <int W>
__device__ __forceinline__ uint32_t tile_off(int row, int piece) {
    static_assert(W == 32 || W == 64 || W == 128, "tile width");
    if (W == 32) return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
    return (uint32_t)(row * (W * 2) + ((piece ^ (row & 7)) << 4));
}

// B operand for two 8-column blocks, B[k][n] = tile[n][k]: rows n0 .. n0 + 15, pieces 2 kk, 2 kk + 1.
// r[0], r[1]: the first block's; r[2], r[3]: the second's.
template <int W>
__device__ __forceinline__ void b_rows(uint32_t (&r)[4], uint32_t tile, int n0, int kk, int lane) {
    const int m = lane >> 3;
    ldm(r, tile + tile_off<W>(n0 + ((m >> 1) << 3) + (lane & 7), 2 * kk + (m & 1)));
}
// B[k][n] = tile[k][n]: rows k0 .. k0 + 15, columns 16 np .. 16 np + 15.
template <int W>
__device__ __forceinline__ void b_cols(uint32_t (&r)[4], uint32_t tile, int k0, int np, int lane) {
    const int m = lane >> 3;
    ldm_t(r, tile + tile_off<W>(k0 + ((m & 1) << 3) + (lane & 7), 2 * np + (m >> 1)));
}
// A[m][k] = tile[m][k]: rows m0 .. m0 + 15, pieces 2 kk, 2 kk + 1.
template <int W>
__device__ __forceinline__ void a_rows(uint32_t (&r)[4], uint32_t tile, int m0, int kk, int lane) {
    const int m = lane >> 3;
    ldm(r, tile + tile_off<W>(m0 + ((m & 1) << 3) + (lane & 7), 2 * kk + (m >> 1)));
}
// A[m][k] = tile[k][m]: rows k0 .. k0 + 15, columns 16 mp .. 16 mp + 15.
template <int W>
__device__ __forceinline__ void a_cols(uint32_t (&r)[4], uint32_t tile, int k0, int mp, int lane) {
    const int m = lane >> 3;
    ldm_t(r, tile + tile_off<W>(k0 + ((m >> 1) << 3) + (lane & 7), 2 * mp + (m & 1)));
}

// Block (ib, jb) of a lower triangular 64 x 64 matrix kept as 16 x 16 blocks of
// four 8 x 8 matrices (128 bytes each, order: row half, column half).
__device__ __forceinline__ int tri(int ib, int jb) { return (ib * (ib + 1) >> 1) + jb; }

// ---- gates of one chunk
using Gates = DeltaGates;

// 2^x to 2 units in the last place, denormal results as 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// G_ij for row i (its gh, gl) and columns j, j + 1; `keep`: the largest column that counts,
// the others are 0 (their exponent may overflow, so they are selected away, not multiplied).
__device__ __forceinline__ float2 gamma_pair(float gh, float gl, const Gates& s, int j, int keep) {
    const float2 h = *reinterpret_cast<const float2*>(&s.gh[j]), l = *reinterpret_cast<const float2*>(&s.gl[j]);
    const float x = exp2_fast((gh - h.x) + (gl - l.x)), y = exp2_fast((gh - h.y) + (gl - l.y));
    return make_float2(j <= keep ? x : 0.f, j + 1 <= keep ? y : 0.f);
}
__device__ __forceinline__ float select0(bool on, float x) { return on ? x : 0.f; }

// Forms the gates of tokens n0 .. n0 + 63 (one warp, every lane).
__device__ __forceinline__ void form_gates(Gates& s, const DeltaParams& p, int b, int h, int n0, int lane) {
    double g[2];
    float be[2];
    int lv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int n = n0 + 2 * lane + i;
        lv[i] = n < p.N && (!p.mask || p.mask[(int64_t)b * p.mask_sb + n] != 0);
        be[i] = 0.f;
        g[i] = 0.0;
        if (lv[i]) {
            be[i] = p.beta.p ? p.beta.p[b * p.beta.sb + h * p.beta.sh + n * p.beta.sn] : 1.f;
            if (p.lg.p) {
                const float x = p.lg.p[b * p.lg.sb + h * p.lg.sh + n * p.lg.sn];
                g[i] = x < kMinLogGamma ? kMinLogGamma : x;
            }
        }
    }
    double run = g[0] + g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
    }
    const double total = __shfl_sync(0xffffffffu, run, 31);
    const int any = __any_sync(0xffffffffu, lv[0] | lv[1]), full = __all_sync(0xffffffffu, lv[0] & lv[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double gi = i ? run : run - g[1];
        const int t = 2 * lane + i;
        const double g2 = gi * 1.4426950408889634;  // 1 / ln 2
        const float hi = (float)g2;
        s.gh[t] = hi;
        s.gl[t] = (float)(g2 - (double)hi);
        s.beta[t] = be[i];
        s.eg[t] = expf((float)gi);
        s.kd[t] = expf((float)(total - gi));
        s.live[t] = lv[i];
    }
    if (lane == 0) {
        s.eC = expf((float)total);
        s.dC = expm1f((float)total);
        s.any = any;
        s.full = full;
    }
}

// ---- [64][W] tiles from global memory, through registers
// A tile's 16-byte pieces (8 elements) in the registers of NT threads, between
// the load (issue) and, an iteration later, the store to shared memory: masked
// rows are zeroed there, whatever memory holds.
template <typename T, int W, int NT>
struct TileRegs {
    static constexpr int kPieces = W / 8, kPer = 64 * kPieces / NT, kQ = sizeof(T) / 2, kRows = NT / kPieces;
    static_assert(64 * kPieces % NT == 0, "threads per tile");
    uint4 r[kPer][kQ];

    __device__ __forceinline__ void issue(const DeltaTensor& x, int64_t base, int n0, int c0, int width, int N, int tid) {
        const int c = c0 + tid % kPieces * 8, n1 = n0 + tid / kPieces;
        const T* src = static_cast<const T*>(x.p) + base + n1 * x.sn + c;
        if (x.vec && width % 8 == 0) {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const bool in = n1 + u * kRows < N && c < width;
#pragma unroll
                for (int i = 0; i < kQ; ++i)
                    r[u][i] = in ? __ldg(reinterpret_cast<const uint4*>(src + u * kRows * x.sn) + i) : make_uint4(0, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                alignas(16) T t[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    t[i] = n1 + u * kRows < N && c + i < width ? src[u * kRows * x.sn + i] : from_f<T>(0.f);
#pragma unroll
                for (int i = 0; i < kQ; ++i) r[u][i] = reinterpret_cast<const uint4*>(t)[i];
            }
        }
    }

    __device__ __forceinline__ void values(int u, float (&f)[8]) const {
        if constexpr (kQ == 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[4 * i] = __uint_as_float(r[u][i].x);
                f[4 * i + 1] = __uint_as_float(r[u][i].y);
                f[4 * i + 2] = __uint_as_float(r[u][i].z);
                f[4 * i + 3] = __uint_as_float(r[u][i].w);
            }
        } else {
            const uint32_t w[4] = {r[u][0].x, r[u][0].y, r[u][0].z, r[u][0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                T t[2];
                *reinterpret_cast<uint32_t*>(t) = w[i];
                f[2 * i] = to_f<T>(t[0]);
                f[2 * i + 1] = to_f<T>(t[1]);
            }
        }
    }

    // as NP bf16 planes of [64][W]
    template <int NP>
    __device__ __forceinline__ void store_planes(unsigned char* tile, const int* live, int tid) const {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int idx = tid + u * NT, row = idx / kPieces, piece = idx % kPieces;
            unsigned char* at = tile + tile_off<W>(row, piece);
            const bool on = live[row] != 0;
            if constexpr (NP == 1) {
                *reinterpret_cast<uint4*>(at) = on ? r[u][0] : make_uint4(0, 0, 0, 0);
            } else {
                float f[8];
                values(u, f);
                uint32_t q[4][NP];
#pragma unroll
                for (int i = 0; i < 4; ++i) split2<NP>(on ? f[2 * i] : 0.f, on ? f[2 * i + 1] : 0.f, q[i]);
#pragma unroll
                for (int pl = 0; pl < NP; ++pl)
                    *reinterpret_cast<uint4*>(at + pl * (64 * W * 2)) = make_uint4(q[0][pl], q[1][pl], q[2][pl], q[3][pl]);
            }
        }
    }
};

// A tile loaded and stored at once, a few pieces at a time.
template <typename T, int W, int NP, int NT>
__device__ __forceinline__ void load_tile(unsigned char* tile, const DeltaTensor& x, int64_t base, int n0, int c0, int width, int N,
                                          const int* live, int tid) {
    TileRegs<T, W, NT> r;
    r.issue(x, base, n0, c0, width, N, tid);
    r.template store_planes<NP>(tile, live, tid);
}

// BYTES contiguous bytes (a multiple of 16) the same way.
template <int BYTES, int NT>
struct ByteRegs {
    static constexpr int kPer = (BYTES / 16 + NT - 1) / NT;
    uint4 r[kPer];
    __device__ __forceinline__ void issue(const void* src, int tid) {
#pragma unroll
        for (int u = 0; u < kPer; ++u)
            if (tid + u * NT < BYTES / 16) r[u] = __ldg(static_cast<const uint4*>(src) + tid + u * NT);
    }
    __device__ __forceinline__ void store(void* dst, int tid) const {
#pragma unroll
        for (int u = 0; u < kPer; ++u)
            if (tid + u * NT < BYTES / 16) static_cast<uint4*>(dst)[tid + u * NT] = r[u];
    }
};

// NT threads start BYTES contiguous bytes on their way to shared memory.
template <int NT>
__device__ __forceinline__ void async16(unsigned char* dst, const unsigned char* src, int bytes, int tid) {
    for (int i = tid * 16; i < bytes; i += NT * 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst + i)), "l"(src + i) : "memory");
}
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last N groups have arrived.
template <int N>
__device__ __forceinline__ void async_wait_but() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A [64][W] tile of 16-bit elements straight to shared memory (one plane); rows from N and columns from `width`
// (a multiple of 8) are zero, masked rows hold what memory holds (clear_dead removes it). Rows start on 16 bytes.
template <typename T, int W, int NT>
__device__ __forceinline__ void async_tile(unsigned char* tile, const DeltaTensor& x, int64_t base, int n0, int c0, int width, int N,
                                           int tid) {
    constexpr int kPieces = W / 8, kPer = 64 * kPieces / NT, kRows = NT / kPieces;
    const int piece = tid % kPieces, row = tid / kPieces, c = c0 + piece * 8;
    const T* src = static_cast<const T*>(x.p) + base + (n0 + row) * x.sn + c;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
        const bool in = n0 + row + u * kRows < N && c < width;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(tile + tile_off<W>(row + u * kRows, piece))),
                     "l"(in ? src + u * kRows * x.sn : static_cast<const T*>(x.p)), "r"(in ? 16 : 0)
                     : "memory");
    }
}
template <int W, int NT>
__device__ __forceinline__ void clear_dead(unsigned char* tile, const int* live, int tid) {
    constexpr int kPieces = W / 8;
    for (int i = tid; i < 64 * kPieces; i += NT)
        if (!live[i / kPieces]) *reinterpret_cast<uint4*>(tile + tile_off<W>(i / kPieces, i % kPieces)) = make_uint4(0, 0, 0, 0);
}

template <int NT>
__device__ __forceinline__ void copy16(unsigned char* dst, const unsigned char* src, int bytes, int tid) {
    for (int i = tid * 16; i < bytes; i += NT * 16)
        *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(src + i);
}

// What one CTA of a walk has to do: chunks [begin, end) of a sequence, 32 columns from c0.
struct WalkJob {
    int64_t bh;
    int b, h, begin, end, cb, c0;
    bool ident;        // columns of the identity (V = 0) in place of value columns: the walk then gives seg_M's columns
    const float* in;   // state before, [d, ld], or null (0)
    float* out;        // state after, or null
    int ld, rows;      // of `in` and `out`
};

__device__ __forceinline__ int64_t tensor_base(const DeltaTensor& x, int b, int h) {
    return b * x.sb + (x.group == 1 ? h : h / x.group) * x.sh;
}

// scale G o (Q K^T) for row block rb, as NX planes in `out`
// (10 lower triangular blocks per plane).
template <int DP, int NIN, int NX>
__device__ __forceinline__ void score_rows(unsigned char* out, uint32_t q, uint32_t k, const Gates& s, float scale, int rb, int lane) {
    constexpr int kTile = 64 * DP * 2;
    float acc[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
#pragma unroll 2
    for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t a[NIN][4];
#pragma unroll
        for (int pl = 0; pl < NIN; ++pl) a_rows<DP>(a[pl], q + pl * kTile, 16 * rb, kk, lane);
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
            if (jb <= rb) {
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
    }
    const int g = lane >> 2, t = lane & 3, i0 = 16 * rb + g;
    const float gh[2] = {s.gh[i0], s.gh[i0 + 8]}, gl[2] = {s.gl[i0], s.gl[i0 + 8]};
#pragma unroll
    for (int jb = 0; jb < 4; ++jb) {
        if (jb > rb) continue;
        unsigned char* blk = out + tri(rb, jb) * 512 + lane * 4;
#pragma unroll
        for (int jh = 0; jh < 2; ++jh) {
            const int j = 16 * jb + 8 * jh + 2 * t;
#pragma unroll
            for (int ih = 0; ih < 2; ++ih) {
                const float2 ga = gamma_pair(gh[ih], gl[ih], s, j, i0 + 8 * ih);
                uint32_t r[NX];
                split2<NX>(scale * ga.x * select0(j <= i0 + 8 * ih, acc[2 * jb + jh][2 * ih]),
                           scale * ga.y * select0(j + 1 <= i0 + 8 * ih, acc[2 * jb + jh][2 * ih + 1]), r);
#pragma unroll
                for (int pl = 0; pl < NX; ++pl)
                    *reinterpret_cast<uint32_t*>(blk + pl * (kYBlocks * 512) + (ih * 2 + jh) * 128) = r[pl];
            }
        }
    }
}

// The two warps of a pair share a chunk's four blocks of 16 tokens so that both have half of a triangle's blocks:
// warp 0 has blocks 0 and 3, warp 1 has 1 and 2. (One code for both: the blocks are run-time values, so that the
// walks' loops stay small enough for the instruction cache.)
struct Own {
    int b0, b1;
    __device__ explicit Own(int a) : b0(a ? 1 : 0), b1(a ? 2 : 3) {}
    __device__ int at(int u) const { return u ? b1 : b0; }
};

template <int NB>
__device__ __forceinline__ void zero_acc(float (&c)[NB][4]) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
}
// The state after a chunk: e^{g_C} S + the chunk's part U. (Products added to S itself would each cut it off towards zero:
// 256 chunks without decay were 8e-5 off in float32, 5e-5 in bf16. An e^{g_C} near 1 that is rounded by itself is off by
// up to 2^-25, the same way at every chunk of a constant decay: 256 chunks 7.6e-6.)
template <int NB>
__device__ __forceinline__ void next_state(float (&S)[NB][4], const Gates& s, const float (&U)[NB][4]) {
    const float eC = s.eC, dC = s.dC;
    if (fabsf(dC) < 0.0625f) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[n][i] += fmaf(dC, S[n][i], U[n][i]);
    } else {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[n][i] = fmaf(eC, S[n][i], U[n][i]);
    }
}
__device__ __forceinline__ void add_acc(float (&c)[4], float4 x) {
    c[0] += x.x; c[1] += x.y; c[2] += x.z; c[3] += x.w;
}
__device__ __forceinline__ float4 as_float4(const float (&c)[4]) { return make_float4(c[0], c[1], c[2], c[3]); }

// An accumulator tile (NB blocks of 16 rows x 8 columns) through shared memory, 16 bytes per lane and block.
template <int NB>
__device__ __forceinline__ void put_acc(float4* at, const float (&c)[NB][4], int lane) {
#pragma unroll
    for (int n = 0; n < NB; ++n) at[n * 32 + lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
}
// The planes of an A operand (16 x 16) through shared memory, 16 bytes per lane and plane.
template <int NX>
__device__ __forceinline__ void put_a(unsigned char* tile, const uint32_t (&a)[NX][4], int lane) {
#pragma unroll
    for (int pl = 0; pl < NX; ++pl)
        *reinterpret_cast<uint4*>(tile + pl * 512 + lane * 16) = make_uint4(a[pl][0], a[pl][1], a[pl][2], a[pl][3]);
}
template <int NX>
__device__ __forceinline__ void get_a(uint32_t (&a)[NX][4], const unsigned char* tile, int lane) {
#pragma unroll
    for (int pl = 0; pl < NX; ++pl) {
        const uint4 x = *reinterpret_cast<const uint4*>(tile + pl * 512 + lane * 16);
        a[pl][0] = x.x; a[pl][1] = x.y; a[pl][2] = x.z; a[pl][3] = x.w;
    }
}
// The values that an A operand's planes stand for, as two accumulator blocks.
template <int NX>
__device__ __forceinline__ void from_a(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NX][4]) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        float2 x = unpack_bf16(a[NX - 1][m]);
#pragma unroll
        for (int pl = NX - 2; pl >= 0; --pl) {
            const float2 y = unpack_bf16(a[pl][m]);
            x.x += y.x;
            x.y += y.y;
        }
        float(&c)[4] = m < 2 ? c0 : c1;
        c[2 * (m & 1)] = x.x;
        c[2 * (m & 1) + 1] = x.y;
    }
}
// Two neighbouring float32 accumulator blocks from shared memory.
__device__ __forceinline__ void get_acc2(float (&c0)[4], float (&c1)[4], const float4* at, int lane) {
    const float4 x = at[lane], y = at[32 + lane];
    c0[0] = x.x; c0[1] = x.y; c0[2] = x.z; c0[3] = x.w;
    c1[0] = y.x; c1[1] = y.y; c1[2] = y.z; c1[3] = y.w;
}
// Products of one A operand with 16 rows n0 .. and 16 rows n1 .. of a tile (B[k][n] = tile[n][k]), k block kk.
template <int W, int NA, int NB, int NX>
__device__ __forceinline__ void mma_rows(float (&c)[4][4], const uint32_t (&a)[NA][4], uint32_t tile, int n0, int n1, int kk, int lane) {
    uint32_t b[4][NB][2];
#pragma unroll
    for (int pl = 0; pl < NB; ++pl) {
        uint32_t r[4], q[4];
        b_rows<W>(r, tile + pl * (64 * W * 2), n0, kk, lane);
        b_rows<W>(q, tile + pl * (64 * W * 2), n1, kk, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i >> 1][pl][i & 1] = r[i], b[2 + (i >> 1)][pl][i & 1] = q[i];
    }
    mma_set<4, NA, NB, NX>(c, a, b);
}
// B[k][n] = tile[k][n]: rows k0 .., columns 8 n0 .. 8 (n0 + N) - 1.
template <int N, int W, int NA, int NB, int NX>
__device__ __forceinline__ void mma_cols(float (&c)[N][4], const uint32_t (&a)[NA][4], uint32_t tile, int k0, int n0, int lane) {
    uint32_t b[N][NB][2];
#pragma unroll
    for (int np = 0; np < N / 2; ++np)
#pragma unroll
        for (int pl = 0; pl < NB; ++pl) {
            uint32_t r[4];
            b_cols<W>(r, tile + pl * (64 * W * 2), k0, n0 / 2 + np, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[2 * np + (i >> 1)][pl][i & 1] = r[i];
        }
    mma_set<N, NA, NB, NX>(c, a, b);
}
// B = a 16 x 16 block M[r][c] kept as four 8 x 8 matrices (row half, column half) per plane, planes kYBlocks blocks
// apart; `block` is its address plus lane * 16. KROWS: B[k][n] = M[k][n], else B[k][n] = M[n][k].
template <int NX, bool KROWS>
__device__ __forceinline__ void load_block(uint32_t (&b0)[NX][2], uint32_t (&b1)[NX][2], uint32_t block) {
#pragma unroll
    for (int pl = 0; pl < NX; ++pl) {
        uint32_t r[4];
        if (KROWS) {
            ldm_t(r, block + pl * (kYBlocks * 512));
            b0[pl][0] = r[0]; b0[pl][1] = r[2]; b1[pl][0] = r[1]; b1[pl][1] = r[3];
        } else {
            ldm(r, block + pl * (kYBlocks * 512));
            b0[pl][0] = r[0]; b0[pl][1] = r[1]; b1[pl][0] = r[2]; b1[pl][1] = r[3];
        }
    }
}
// c[0], c[1] += A M0 where `first`, c[2], c[3] += A M1 where `second`.
template <int NA, int NX, bool KROWS>
__device__ __forceinline__ void mma_blocks(float (&c)[4][4], const uint32_t (&a)[NA][4], bool first, uint32_t m0, bool second, uint32_t m1) {
    uint32_t b[4][NX][2];
    if (first && second) {
        load_block<NX, KROWS>(b[0], b[1], m0);
        load_block<NX, KROWS>(b[2], b[3], m1);
        mma_set<4, NA, NX, NX>(c, a, b);
    } else if (first) {
        load_block<NX, KROWS>(b[0], b[1], m0);
        mma_pair<NA, NX, NX>(c[0], c[1], a, b[0], b[1]);
    } else {
        load_block<NX, KROWS>(b[2], b[3], m1);
        mma_pair<NA, NX, NX>(c[2], c[3], a, b[2], b[3]);
    }
}

// Two neighbouring blocks as the planes of an A operand, to memory as four 8 x 8 matrices of 128 bytes per plane.
template <int NX>
__device__ __forceinline__ void store_matrices(unsigned char* dst, const uint32_t (&a)[NX][4], int lane) {
#pragma unroll
    for (int pl = 0; pl < NX; ++pl)
#pragma unroll
        for (int m = 0; m < 4; ++m) *reinterpret_cast<uint32_t*>(dst + pl * 512 + m * 128 + lane * 4) = a[pl][m];
}

}  // namespace dl
}  // namespace subq
