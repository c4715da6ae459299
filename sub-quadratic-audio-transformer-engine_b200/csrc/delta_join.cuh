// Segments of a sequence that are walked side by side: the states between them (see delta_common.cuh).
#pragma once

#include "delta_common.cuh"

namespace subq {
namespace {

using namespace dl;

// seg_S[s] <- M_s S_s + seg_S[s] (what segment s makes of the state before it, S_s), s in order: seg_S[s - 1] is then the
// state before segment s. (The first segment's own state already holds what came before it: its walk started from the
// initial state.) The walk back over the chunks does the same from the last segment to the first: there s counts from the
// end, S is the state's gradient, and M_s the transpose of what the forward has. seg_M holds M_s^T. A CTA has 16 columns of one sequence, a thread four rows of two of them, so that two
// loads from shared memory feed eight multiplications; the operands of the next segments (three, two above d = 64) are on
// their way while one is computed (about 1 us a segment at d = 64; 8 us where each waited for its own).
template <int DP>
struct JoinSmem {
    static constexpr int kThreads = 2 * DP, kBufs = DP == 64 ? 4 : 3;
    alignas(16) float M[kBufs][DP * DP];  // [DP][DP], transposed
    float S[2][DP * 16];
};
template <int DP>
__global__ void __launch_bounds__(2 * DP) delta_join_kernel(const DeltaParams p) {
    constexpr int kThreads = JoinSmem<DP>::kThreads, kBufs = JoinSmem<DP>::kBufs, kAhead = kBufs - 1;
    extern __shared__ __align__(128) unsigned char raw[];
    JoinSmem<DP>& sm = *reinterpret_cast<JoinSmem<DP>*>(raw);
    const unsigned ncb = (p.e + 15) / 16, bh32 = blockIdx.x / ncb;
    const int64_t slot = (int64_t)bh32 * (p.nseg - 1);
    const int tid = threadIdx.x, r0 = tid / 8 * 4, cl = tid % 8 * 2, c = (int)(blockIdx.x - bh32 * ncb) * 16 + cl, last = p.nseg - 2;
    auto send = [&](int s) {
        if (s <= last) async16<kThreads>(reinterpret_cast<unsigned char*>(sm.M[s % kBufs]),
                                         reinterpret_cast<const unsigned char*>(p.seg_M + (slot + s) * (DP * DP)), DP * DP * 4, tid);
        async_commit();
    };
    auto load = [&](float (&l)[4][2], int s) {
        const float* add = p.seg_S + (slot + s) * p.d * p.e + c;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) l[i][j] = s <= last && r0 + i < p.d && c + j < p.e ? add[(r0 + i) * p.e + j] : 0.f;
    };
    for (int s = 1; s <= kAhead; ++s) send(s);
    float l[4][2], next[4][2], after[4][2];
    load(l, 0);
    load(next, 1);
    load(after, 2);
    if (p.seg_in) {
        const int64_t at = (int64_t)bh32 * p.d * p.e + c;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (r0 + i < p.d && c + j < p.e) p.seg_in[at + (r0 + i) * p.e + j] = p.S_in[at + (r0 + i) * p.e + j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(&sm.S[0][(r0 + i) * 16 + cl]) = make_float2(l[i][0], l[i][1]);
    for (int s = 1; s <= last; ++s) {
        const float* M = sm.M[s % kBufs];
        const float* S = sm.S[(s - 1) & 1];
        float acc[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = next[i][j], next[i][j] = after[i][j];
        async_wait_but<kAhead - 1>();  // this thread's pieces of M_s
        __syncthreads();               // everyone's, and S; M_{s - 1} has been read
        send(s + kAhead);
        load(after, s + 2);
        // (rows and columns from d: S is 0 there, and M, the identity's columns that were walked, finite; columns of M
        // that were not walked are left out by the bound)
        const int end = (p.d + 31) / 32 * 32;
#pragma unroll 8
        for (int x = 0; x < end; ++x) {
            const float4 w = *reinterpret_cast<const float4*>(&M[x * DP + r0]);
            const float2 v = *reinterpret_cast<const float2*>(&S[x * 16 + cl]);
            acc[0][0] = fmaf(w.x, v.x, acc[0][0]); acc[0][1] = fmaf(w.x, v.y, acc[0][1]);
            acc[1][0] = fmaf(w.y, v.x, acc[1][0]); acc[1][1] = fmaf(w.y, v.y, acc[1][1]);
            acc[2][0] = fmaf(w.z, v.x, acc[2][0]); acc[2][1] = fmaf(w.z, v.y, acc[2][1]);
            acc[3][0] = fmaf(w.w, v.x, acc[3][0]); acc[3][1] = fmaf(w.w, v.y, acc[3][1]);
        }
        float* out = p.seg_S + (slot + s) * p.d * p.e + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool row = r0 + i < p.d, in[2] = {row && c < p.e, row && c + 1 < p.e};
            *reinterpret_cast<float2*>(&sm.S[s & 1][(r0 + i) * 16 + cl]) = make_float2(in[0] ? acc[i][0] : 0.f, in[1] ? acc[i][1] : 0.f);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (in[j]) out[(r0 + i) * p.e + j] = acc[i][j];
        }
    }
    async_wait();
}

template <int DP>
cudaError_t join_t(const DeltaParams& p, cudaStream_t st) {
    const int smem = (int)sizeof(JoinSmem<DP>);
    const cudaError_t err = cudaFuncSetAttribute(delta_join_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    delta_join_kernel<DP><<<(unsigned)((int64_t)p.B * p.H * ((p.e + 15) / 16)), JoinSmem<DP>::kThreads, smem, st>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace subq
