// Matrix product of e4m3 operands with a float32 scale for every 1 x 128 of a and every 128 x 128 of b:
//   out[m, n] = bias[n] + sum_kb a_scale[m, kb] b_scale[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k].
//
// Tensor-core kernels: one thread loads the 128-byte rows of a k-block of both operands by TMA (zeros behind the last row and
// column), one issues its four tcgen05.mma (kind::f8f6f4, K = 32 each) into one of two TMEM accumulators, and the epilogue's
// warps read the finished one back, row m in lane m, multiply it by the block's two scales and add it to float32 sums in
// registers, while the other accumulator is being formed: a scale for every k-block is a rounding of 24 bits, and what the
// tensor core adds up by itself is 128 products.
//
// Large products: 128 x 256 tiles by one CTA an SM that goes on from tile to tile (k-blocks of the next one are loaded and
// multiplied while this one is written), eight epilogue warps with 128 columns each. A k-block's products take 512 cycles,
// its way through the epilogue (TMEM read and multiply-add, two warps to a scheduler) about as long, its 48 KB from L2 about
// 800: 16384 x 4096 x 1024 takes 107 to 118 us from card to card (1.2 to 1.3 PFLOP/s), 2048 x 4096 x 4096 51 us (1.35). That is 1600
// cycles a k-block at K = 1024: beside L2 the stores of a finished tile, during which two more k-blocks at most are formed.
// Smaller ones: 128 x BN tiles, a CTA each, two to an SM.
// A few rows (streaming steps) are bound by the weights' bytes, or by the launch: there a warp has a column of b, its lanes
// 16 values each at a time, and every row of a.
#include <cuda_fp8.h>

#include "block_launch.h"
#include "sel_common.cuh"
#include "tc_common.cuh"

namespace subq {
namespace {

using sel::F2;
using sel::f2;

constexpr int kBM = 128, kBK = 128;

template <typename T, int BN>
struct MatmulShape {
    static constexpr int kStages = BN >= 128 ? 3 : 4;
    static constexpr int kABytes = kBM * kBK, kBBytes = BN * kBK, kStageBytes = kABytes + kBBytes;
    static constexpr int kPad = 16 / (int)sizeof(T);  // elements between two rows of the staged outputs, against bank conflicts
    static constexpr int kOutBytes = kBM * (BN + kPad) * (int)sizeof(T);
    static constexpr int kTiles = kStages * kStageBytes > kOutBytes ? kStages * kStageBytes : (kOutBytes + 1023) / 1024 * 1024;
    static constexpr int kSmem = kTiles + 1024;  // (aligned to 1024 inside)
    static constexpr int kTmemCols = 2 * BN;
    static constexpr int kThreads = 192;
};

template <typename T, int BN>
__global__ void __launch_bounds__(192, 2) scaled_matmul_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                                                               const MatmulParams p) {
    using S = MatmulShape<T, BN>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    unsigned char* smem = raw + (1024 - (tc::smem_u32(raw) & 1023)) % 1024;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntiles = (p.N + BN - 1) / BN;
    const int64_t m0 = (int64_t)(blockIdx.x / ntiles) * kBM;
    const int n0 = (int)(blockIdx.x % ntiles) * BN;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_empty[i], 4);
        }
        tc::fence_mbar_init();
    }
    if (warp == 5) tc::tmem_alloc(&tmem_slot, S::kTmemCols);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    if (warp == 4) {
        if (lane == 0) {
            int issued = 0;
            for (int kb = 0; kb < p.nk && ok; ++kb) {
                const int s = kb % S::kStages;
                if (kb >= S::kStages) ok = tcs::wait_bar(&empty[s], (kb / S::kStages - 1) & 1, p.status);
                if (!ok) break;
                unsigned char* at = smem + s * S::kStageBytes;
                tc::mbar_arrive_expect_tx(&full[s], S::kStageBytes);
                tc::tma_load_2d(at, &ta, kb * kBK, (int)m0, &full[s]);
                tc::tma_load_2d(at + S::kABytes, &tb, kb * kBK, n0, &full[s]);
                ++issued;
            }
            if (!ok)  // the copies in flight land before the CTA ends
                for (int kb = issued > S::kStages ? issued - S::kStages : 0; kb < issued; ++kb) tcs::wait_bar(&full[kb % S::kStages], (kb / S::kStages) & 1, p.status);
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc_e4m3(kBM, BN);
            const uint32_t base = tc::smem_u32(smem);
            int issued = 0;
            for (int kb = 0; kb < p.nk && ok; ++kb) {
                const int s = kb % S::kStages, buf = kb & 1;
                ok = tcs::wait_bar(&full[s], (kb / S::kStages) & 1, p.status);
                if (ok && kb >= 2) ok = tcs::wait_bar(&acc_empty[buf], (kb / 2 - 1) & 1, p.status);
                if (!ok) break;
                tc::tc_fence_after();
                const uint64_t ad = tc::sdesc_sw128(base + s * S::kStageBytes, 0, 1024), bd = tc::sdesc_sw128(base + s * S::kStageBytes + S::kABytes, 0, 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_f8(tmem + buf * BN, ad + 2 * k, bd + 2 * k, id, k > 0);
                tc::mma_commit(&empty[s]);
                tc::mma_commit(&acc_full[buf]);
                ++issued;
            }
            if (!ok && issued) tcs::wait_bar(&acc_full[(issued - 1) & 1], ((issued - 1) / 2) & 1, p.status);
        }
        __syncwarp();
    } else {
        const int row = warp * 32 + lane;
        const int64_t m = m0 + row;
        const bool in = m < p.M;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        float acc[BN];
#pragma unroll
        for (int i = 0; i < BN; ++i) acc[i] = 0.f;
        const float* as = p.a_scale + (in ? m : 0) * p.as_s;
        const float* bs = p.b_scale + (int64_t)(n0 / 128) * p.bs_s;
        float sa = as[0], sb = bs[0];
        for (int kb = 0; kb < p.nk; ++kb) {
            const int buf = kb & 1;
            const float scale = in ? sa * sb : 0.f;
            if (kb + 1 < p.nk) {
                sa = as[kb + 1];
                sb = bs[kb + 1];
            }
            ok = __all_sync(0xffffffffu, tcs::wait_bar(&acc_full[buf], (kb / 2) & 1, p.status));
            if (!ok) break;
            tc::tc_fence_after();
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                tc::tmem_ld32_issue(tmem + buf * BN + c + lanes, v);
                tc::tmem_wait_ld();
                tc::tmem_regs_ready<32>(v);
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(__uint_as_float(v[i]), scale, acc[c + i]);
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
        }
        // Every product has been read back, so the stages are free: a warp's 32 rows go through them to rows that are
        // written whole.
        if (ok) {
            T* stage = reinterpret_cast<T*>(smem) + (size_t)warp * 32 * (BN + S::kPad);
            T* mine = stage + lane * (BN + S::kPad);
            constexpr int kV = 16 / (int)sizeof(T), kPer = BN / kV;  // 16-byte pieces of a row
#pragma unroll
            for (int c = 0; c < BN; c += kV) {
                sel::Piece<T, kV> o;
#pragma unroll
                for (int i = 0; i < kV; ++i) o.x[i] = from_f<T>(p.bias && n0 + c + i < p.N ? acc[c + i] + p.bias[n0 + c + i] : acc[c + i]);
                o.store(mine + c);
            }
            __syncwarp();
            const bool vec = n0 + BN <= p.N && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_s * (int64_t)sizeof(T) % 16 == 0;
            T* out = static_cast<T*>(p.out);
            const int64_t mw = m0 + warp * 32;
            if (vec) {
                for (int i = lane; i < 32 * kPer; i += 32) {
                    const int r = i / kPer, c = i % kPer * kV;
                    if (mw + r < p.M) *reinterpret_cast<uint4*>(out + (mw + r) * p.out_s + n0 + c) = *reinterpret_cast<const uint4*>(stage + r * (BN + S::kPad) + c);
                }
            } else {
                for (int i = lane; i < 32 * BN; i += 32) {
                    const int r = i / BN, c = i % BN;
                    if (mw + r < p.M && n0 + c < p.N) out[(mw + r) * p.out_s + n0 + c] = stage[r * (BN + S::kPad) + c];
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 5) tc::tmem_dealloc(tmem, S::kTmemCols);
}

// ------------------------------------------------------------------ 128 x 256 tiles, one CTA an SM
template <typename T>
struct BigShape {
    static constexpr int kBN = 256, kStages = 4, kABytes = kBM * kBK, kStageBytes = kABytes + kBN * kBK;
    static constexpr int kRow = 64 + 16;              // bytes of a staged output row, against bank conflicts
    static constexpr int kOut = 8 * 32 * kRow;         // eight warps' 32 rows
    static constexpr int kSmem = kStages * kStageBytes + kOut + 1024;
    static constexpr int kThreads = 384;  // two warpgroups for the epilogue, one whose first two warps load and multiply
};

template <typename T>
__global__ void __launch_bounds__(384, 1) scaled_matmul_big_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const MatmulParams p,
                                                                   int64_t tiles, int ntiles) {
    using S = BigShape<T>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    unsigned char* smem = raw + (1024 - (tc::smem_u32(raw) & 1023)) % 1024;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_empty[i], 8);
        }
        tc::fence_mbar_init();
    }
    if (warp == 9) tc::tmem_alloc(&tmem_slot, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    // The epilogue's sums and the 64 values that are on their way to them take 200 registers: 256 x 200 + 128 x 104 = 384 x 168 (208 and 88, 216 and 72: 121 us for 107).
    // (k-blocks are counted through all of the CTA's tiles: block i uses stage i % 4 and accumulator i % 2)
    if (warp >= 8) {
    tc::regs_down<104>();
    if (warp == 8) {
        if (lane == 0) {
            int64_t it = 0;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int m0 = (int)(tile / ntiles) * kBM, n0 = (int)(tile % ntiles) * S::kBN;
                for (int kb = 0; kb < p.nk; ++kb, ++it) {
                    const int s = (int)(it % S::kStages);
                    if (it >= S::kStages) ok = tcs::wait_bar(&empty[s], (uint32_t)(it / S::kStages - 1) & 1, p.status);
                    if (!ok) break;
                    unsigned char* at = smem + s * S::kStageBytes;
                    tc::mbar_arrive_expect_tx(&full[s], S::kStageBytes);
                    tc::tma_load_2d(at, &ta, kb * kBK, m0, &full[s]);
                    tc::tma_load_2d(at + S::kABytes, &tb, kb * kBK, n0, &full[s]);
                }
            }
            if (!ok)  // the copies in flight land before the CTA ends
                for (int64_t i = it > S::kStages ? it - S::kStages : 0; i < it; ++i) tcs::wait_bar(&full[i % S::kStages], (uint32_t)(i / S::kStages) & 1, p.status);
        }
        __syncwarp();
    } else if (warp == 9) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc_e4m3(kBM, S::kBN);
            const uint32_t base = tc::smem_u32(smem);
            int64_t it = 0;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x)
                for (int kb = 0; kb < p.nk; ++kb, ++it) {
                    const int s = (int)(it % S::kStages), buf = (int)(it & 1);
                    ok = tcs::wait_bar(&full[s], (uint32_t)(it / S::kStages) & 1, p.status);
                    if (ok && it >= 2) ok = tcs::wait_bar(&acc_empty[buf], (uint32_t)(it / 2 - 1) & 1, p.status);
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint64_t ad = tc::sdesc_sw128(base + s * S::kStageBytes, 0, 1024), bd = tc::sdesc_sw128(base + s * S::kStageBytes + S::kABytes, 0, 1024);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_f8(tmem + buf * S::kBN, ad + 2 * k, bd + 2 * k, id, k > 0);
                    tc::mma_commit(&empty[s]);
                    tc::mma_commit(&acc_full[buf]);
                }
            if (!ok && it) tcs::wait_bar(&acc_full[(it - 1) & 1], (uint32_t)((it - 1) / 2) & 1, p.status);
        }
        __syncwarp();
    }
    } else {
        tc::regs_up<200>();
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        unsigned char* stage = smem + S::kStages * S::kStageBytes + warp * 32 * S::kRow;
        T* out = static_cast<T*>(p.out);
        const bool aligned = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_s * (int64_t)sizeof(T) % 16 == 0;
        int64_t it = 0;
        // scales of a tile's first two k-blocks, asked for before the tile before it is written
        float sa = 0.f, sb = 0.f, sa1 = 0.f, sb1 = 0.f;
        auto begin = [&](int64_t tile, const float*& as, const float*& bs) {
            const int64_t m = tile / ntiles * kBM + quad * 32 + lane;
            const int n0 = (int)(tile % ntiles) * S::kBN + half * 128;
            const bool in = m < p.M && n0 < p.N;
            as = p.a_scale + (in ? m : 0) * p.as_s;
            bs = p.b_scale + (in ? n0 / 128 : 0) * p.bs_s;
            sa = as[0], sb = bs[0];
            if (p.nk > 1) sa1 = as[1], sb1 = bs[1];
        };
        const float *as = nullptr, *bs = nullptr;
        begin(blockIdx.x, as, bs);
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int64_t mw = tile / ntiles * kBM + quad * 32, m = mw + lane;
            const int n0 = (int)(tile % ntiles) * S::kBN + half * 128;
            const bool in = m < p.M && n0 < p.N;
            F2 acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = f2(0.f);
            for (int kb = 0; kb < p.nk; ++kb, ++it) {
                const int buf = (int)(it & 1);
                const F2 scale = f2(in ? sa * sb : 0.f);
                sa = sa1;
                sb = sb1;
                if (kb + 2 < p.nk) {
                    sa1 = as[kb + 2];
                    sb1 = bs[kb + 2];
                }
                ok = __all_sync(0xffffffffu, tcs::wait_bar(&acc_full[buf], (uint32_t)(it / 2) & 1, p.status));
                if (!ok) break;
                tc::tc_fence_after();
                const uint32_t from = tmem + buf * S::kBN + half * 128 + lanes;
                uint32_t v[2][32];  // one half is added while the other is read
                tc::tmem_ld32_issue(from, v[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc::tmem_wait_ld();
                    tc::tmem_regs_ready<32>(v[c & 1]);
                    if (c < 3) {
                        tc::tmem_ld32_issue(from + 32 * (c + 1), v[(c + 1) & 1]);
                    } else {  // everything has been read
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        acc[16 * c + i] = sel::fma(f2(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), scale, acc[16 * c + i]);
                }
            }
            if (!ok) break;
            if (tile + gridDim.x < tiles) begin(tile + gridDim.x, as, bs);
            // 64 bytes of each of the warp's 32 rows at a time, through shared memory to whole sectors of the rows
            constexpr int kC = 64 / (int)sizeof(T), kV = 16 / (int)sizeof(T);
#pragma unroll
            for (int c = 0; c < 128; c += kC) {
                if (n0 + c < p.N) {
#pragma unroll
                    for (int i = 0; i < kC; i += kV) {
                        sel::Piece<T, kV> o;
#pragma unroll
                        for (int k = 0; k < kV; k += 2) {
                            float x, y;
                            sel::get(acc[(c + i + k) / 2], x, y);
                            if (p.bias) {
                                x += n0 + c + i + k < p.N ? p.bias[n0 + c + i + k] : 0.f;
                                y += n0 + c + i + k + 1 < p.N ? p.bias[n0 + c + i + k + 1] : 0.f;
                            }
                            o.x[k] = from_f<T>(x);
                            o.x[k + 1] = from_f<T>(y);
                        }
                        o.store(reinterpret_cast<T*>(stage + lane * S::kRow) + i);
                    }
                    __syncwarp();
                    if (aligned && n0 + c + kC <= p.N) {
#pragma unroll
                        for (int r = lane / 4; r < 32; r += 8)
                            if (mw + r < p.M)
                                *reinterpret_cast<uint4*>(out + (mw + r) * p.out_s + n0 + c + lane % 4 * kV) = *reinterpret_cast<const uint4*>(stage + r * S::kRow + lane % 4 * 16);
                    } else {
                        for (int i = lane; i < 32 * kC; i += 32) {
                            const int r = i / kC, x = i % kC;
                            if (mw + r < p.M && n0 + c + x < p.N) out[(mw + r) * p.out_s + n0 + c + x] = reinterpret_cast<const T*>(stage + r * S::kRow)[x];
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

// 16 values of a row of e4m3 as float32 (zeros behind `left`).
__device__ __forceinline__ void load16(const uint8_t* at, int left, uint4& x) {
    if (left >= 16) {
        x = *reinterpret_cast<const uint4*>(at);
        return;
    }
    uint8_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < left ? at[i] : 0;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[4 * i] | (uint32_t)v[4 * i + 1] << 8 | (uint32_t)v[4 * i + 2] << 16 | (uint32_t)v[4 * i + 3] << 24;
    x = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void to_float16(const uint4& x, float (&f)[16]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}

// MR rows of a, a column of b a warp.
template <typename T, int MR>
__global__ void __launch_bounds__(256) scaled_rows_kernel(const MatmulParams p) {
    const int lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t m0 = (int64_t)blockIdx.y * MR;
    if (n >= p.N) return;
    const uint8_t* b = static_cast<const uint8_t*>(p.b) + (int64_t)n * p.b_s;
    const uint8_t* a = static_cast<const uint8_t*>(p.a) + m0 * p.a_s;
    const float* bs = p.b_scale + (int64_t)(n / 128) * p.bs_s;
    float acc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = 0.f;
#pragma unroll 2
    for (int k = 16 * lane; k < p.K; k += 512) {
        uint4 raw;
        float bf[16];
        load16(b + k, p.K - k, raw);
        to_float16(raw, bf);
        const float sb = bs[k / 128];
#pragma unroll
        for (int r = 0; r < MR; ++r) {
            if (MR > 1 && m0 + r >= p.M) break;
            float af[16], s = 0.f;
            load16(a + r * p.a_s + k, p.K - k, raw);
            to_float16(raw, af);
#pragma unroll
            for (int i = 0; i < 16; ++i) s = fmaf(af[i], bf[i], s);
            acc[r] = fmaf(s, sb * p.a_scale[(m0 + r) * p.as_s + k / 128], acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < MR; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == r && m0 + r < p.M) static_cast<T*>(p.out)[(m0 + r) * p.out_s + n] = from_f<T>(acc[r] + (p.bias ? p.bias[n] : 0.f));
    }
}

template <typename T, int BN>
cudaError_t launch_tiles(MatmulParams p, cudaStream_t st) {
    using S = MatmulShape<T, BN>;
    alignas(64) CUtensorMap ta, tb;
    if (!tcs::make_byte_map(&ta, p.a, p.M, p.K, p.a_s, kBM) || !tcs::make_byte_map(&tb, p.b, p.N, p.K, p.b_s, BN)) return cudaErrorInvalidValue;
    p.status = tcs::status_ptr();
    if (!p.status) return cudaErrorInvalidDevice;
    cudaError_t err = cudaFuncSetAttribute(scaled_matmul_kernel<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = (p.M + kBM - 1) / kBM * ((p.N + BN - 1) / BN);
    scaled_matmul_kernel<T, BN><<<(unsigned)tiles, S::kThreads, S::kSmem, st>>>(ta, tb, p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_big(MatmulParams p, cudaStream_t st) {
    using S = BigShape<T>;
    alignas(64) CUtensorMap ta, tb;
    if (!tcs::make_byte_map(&ta, p.a, p.M, p.K, p.a_s, kBM) || !tcs::make_byte_map(&tb, p.b, p.N, p.K, p.b_s, S::kBN)) return cudaErrorInvalidValue;
    p.status = tcs::status_ptr();
    if (!p.status) return cudaErrorInvalidDevice;
    cudaError_t err = cudaFuncSetAttribute(scaled_matmul_big_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (err != cudaSuccess) return err;
    const int ntiles = (p.N + S::kBN - 1) / S::kBN;
    const int64_t tiles = (p.M + kBM - 1) / kBM * ntiles;
    scaled_matmul_big_kernel<T><<<(unsigned)(tiles < 148 ? tiles : 148), S::kThreads, S::kSmem, st>>>(ta, tb, p, tiles, ntiles);
    return cudaGetLastError();
}

// Device time, us (bf16 out), of the kernels by rows, and of 128 x BN tiles:
//   M, N, K            rows   BN = 32     64    128   256 (persistent)
//   1, 4096, 1024       2.9         -    8.9      -
//   4, 4096, 1024       5.5         -    8.9      -
//   8, 4096, 1024       9.0       8.0    8.8      -
//   8, 4096, 4096      38.1      22.1   22.6      -
//   128, 4096, 1024       -       7.5    8.5    9.1
//   512, 1536, 768        -       7.3    7.4    8.0
//   700, 1000, 2000       -      15.3   15.7   19.0
//   2000, 1000, 2000      -      27.6   18.7   19.7
//   1024, 4096, 1024      -      29.0   18.8   11.9   10.7
//   2048, 4096, 4096      -         -      -     61     51
//   16384, 4096, 1024     -         -      -    140    108
//   5000, 769, 2049       -         -      -     53     78  (fp32 out; the last 256 columns hold one)
// Up to four rows: by rows. Else the narrowest tiles whose CTAs the card holds at once (two an SM); beyond, 128 or 256 columns
// by their waves' times: a wave of two 128 x 128 tiles an SM takes 0.95 of a time in which one of 128 x 256 takes 0.8.
template <typename T>
cudaError_t launch_typed(const MatmulParams& p, cudaStream_t st) {
    if (p.M <= 4 || p.K == 0) {
        const unsigned nb = (unsigned)((p.N + 7) / 8);
        if (p.M == 1) scaled_rows_kernel<T, 1><<<dim3(nb, 1), 256, 0, st>>>(p);
        else scaled_rows_kernel<T, 4><<<dim3(nb, (unsigned)((p.M + 3) / 4)), 256, 0, st>>>(p);
        return cudaGetLastError();
    }
    const int64_t rows = (p.M + kBM - 1) / kBM;
    auto tiles = [&](int bn) { return rows * ((p.N + bn - 1) / bn); };
    if (tiles(32) <= 296) return launch_tiles<T, 32>(p, st);
    if (tiles(64) <= 296) return launch_tiles<T, 64>(p, st);
    return 0.8 * (double)((tiles(256) + 147) / 148) < 0.95 * (double)((tiles(128) + 295) / 296) ? launch_big<T>(p, st) : launch_tiles<T, 128>(p, st);
}

}  // namespace

cudaError_t launch_scaled_matmul(const MatmulParams& p, int out_dtype, cudaStream_t st) {
    return out_dtype == SUBQ_BF16 ? launch_typed<__nv_bfloat16>(p, st) : out_dtype == SUBQ_FP16 ? launch_typed<__half>(p, st) : launch_typed<float>(p, st);
}

}  // namespace subq
