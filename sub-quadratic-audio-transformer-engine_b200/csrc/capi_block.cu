// The C ABI of the selective state space block's operators (include/kernels.hpp): argument checks, workspace, launches.
#include <string.h>

#include <algorithm>

#include "block_launch.h"
#include "capi_common.h"

namespace subq {

#define SUBQ_TYPED(name)                                                                                         \
    cudaError_t name##_bf16(const SelParams& p, SelPass pass, cudaStream_t st);                                  \
    cudaError_t name##_fp16(const SelParams& p, SelPass pass, cudaStream_t st);                                  \
    cudaError_t name##_fp32(const SelParams& p, SelPass pass, cudaStream_t st);                                  \
    cudaError_t name(const SelParams& p, int dtype, SelPass pass, cudaStream_t st) {                             \
        return dtype == SUBQ_BF16 ? name##_bf16(p, pass, st) : dtype == SUBQ_FP16 ? name##_fp16(p, pass, st) : name##_fp32(p, pass, st); \
    }
SUBQ_TYPED(launch_sel_fwd)
SUBQ_TYPED(launch_sel_bwd)
#undef SUBQ_TYPED
#define SUBQ_TYPED(name)                                                                                         \
    cudaError_t name##_bf16(const SelParams& p, cudaStream_t st);                                                \
    cudaError_t name##_fp16(const SelParams& p, cudaStream_t st);                                                \
    cudaError_t name##_fp32(const SelParams& p, cudaStream_t st);                                                \
    cudaError_t name(const SelParams& p, int dtype, cudaStream_t st) {                                           \
        return dtype == SUBQ_BF16 ? name##_bf16(p, st) : dtype == SUBQ_FP16 ? name##_fp16(p, st) : name##_fp32(p, st); \
    }
SUBQ_TYPED(launch_sel_step)
#undef SUBQ_TYPED
cudaError_t launch_sel_sums_bf16(const SelParams& p, bool weights, cudaStream_t st);
cudaError_t launch_sel_sums_fp16(const SelParams& p, bool weights, cudaStream_t st);
cudaError_t launch_sel_sums_fp32(const SelParams& p, bool weights, cudaStream_t st);
cudaError_t launch_sel_sums(const SelParams& p, int dtype, bool weights, cudaStream_t st) {
    return dtype == SUBQ_BF16 ? launch_sel_sums_bf16(p, weights, st) : dtype == SUBQ_FP16 ? launch_sel_sums_fp16(p, weights, st) : launch_sel_sums_fp32(p, weights, st);
}

}  // namespace subq

namespace {

using namespace subq;
using namespace subq::capi;

bool known_type(int dtype) { return dtype == SUBQ_FP32 || dtype == SUBQ_FP16 || dtype == SUBQ_BF16; }

int aligned(const void* p, size_t n, const char* name) {
    return reinterpret_cast<uintptr_t>(p) % n ? fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is not aligned to its element size") : (int)SUBQ_OK;
}

// A [B, L, *] view; `need`: a null pointer is an error.
int tensor3(const subq_tensor3& t, const char* name, int dtype, bool need, SelTensor& out) {
    if (!t.data && need) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    int rc = aligned(t.data, elem_size(dtype), name);
    if (rc) return rc;
    if (t.data && (t.stride_b < 0 || t.stride_l < 0 || t.stride_g < 0)) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
    const uint64_t bytes = (uint64_t)elem_size(dtype);
    const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(t.data) | (uint64_t)t.stride_b * bytes | (uint64_t)t.stride_l * bytes | 16;
    out = {t.data, t.stride_b, t.stride_l, t.stride_g, (int)(all & (~all + 1))};
    return SUBQ_OK;
}

Memory of_rows(const char* name, const SelTensor& t, int64_t B, int64_t L, int64_t G, int64_t width, int dtype) {
    const __int128 es = (__int128)elem_size(dtype);
    return {name, {reinterpret_cast<uintptr_t>(t.p), (int64_t)(width * es), {B, L, G}, {t.sb * es, t.sl * es, t.sg * es}}};
}
Memory of_mask(const uint8_t* mask, int64_t stride, int64_t B, int64_t L) { return {"mask", {reinterpret_cast<uintptr_t>(mask), L, {B, 1, 1}, {stride, 0, 0}}}; }

// -------------------------------------------------------------- selective scan
// Calls of at most this many tokens that fill no handover walk token by token in registers, without shared memory.
constexpr int kSelStepTokens = 8;

int check_sel(const subq_selective_desc& d, SelParams& p) {
    if (d.batch < 0 || d.seq_len < 0 || d.channels < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative batch, seq_len or channels");
    if (d.states <= 0 || d.groups <= 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "states and groups must be positive");
    if (d.states > kSelMaxN) return fail(SUBQ_ERR_UNSUPPORTED, "more than 128 states are not supported");
    if (d.channels % d.groups != 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "groups must be a divisor of channels");
    if (d.batch > 65535 || d.seq_len > (int64_t)1 << 30 || d.channels > (int64_t)1 << 24)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "batch above 65535, seq_len above 2^30 or channels above 2^24");
    if (!known_type(d.dtype)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "the selective scan supports float32, float16 and bfloat16");
    if (d.softplus != 0 && d.softplus != 1) return fail(SUBQ_ERR_INVALID_ARGUMENT, "softplus must be 0 or 1");
    if (d.mask && d.mask_stride_b < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "mask has a negative stride");
    int rc;
    if ((rc = aligned(d.A, 4, "A")) || (rc = aligned(d.D, 4, "D")) || (rc = aligned(d.dt_bias, 4, "dt_bias"))) return rc;
    if (!d.A && d.channels > 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "A is null");
    p = SelParams{};
    p.B = (int)d.batch; p.L = (int)d.seq_len; p.D = (int)d.channels; p.N = (int)d.states; p.G = (int)d.groups;
    p.Dg = p.D / p.G;
    p.softplus = d.softplus;
    p.A = d.A; p.Dw = d.D; p.dt_bias = d.dt_bias;
    p.mask = d.mask;
    p.mask_sb = d.mask ? d.mask_stride_b : 0;
    const int64_t ch = sel_channels(p.N);
    if ((int64_t)p.B * p.G * ((p.Dg + ch - 1) / ch) > 0x7fffffff || (int64_t)p.B * p.D * sel_lanes(p.N) / kSelThreads >= 0x7fffffff)
        return fail(SUBQ_ERR_UNSUPPORTED, "batch * channels is too large for one call");
    p.nseg = 1;
    p.seg_tokens = std::max(kSelTile, (p.L + kSelTile - 1) / kSelTile * kSelTile);
    return SUBQ_OK;
}

// Segments of a sequence that are walked side by side. The walk is bound by instruction issue: an SM with c CTAs takes c times
// a CTA's time (at least 1.6 times: fewer warps than that leave it waiting), so what counts is how evenly the grid fills the
// SMs. A segment costs `first` of the walk again for its sum in the launch before, 4 us for that launch, and a step of the
// chain in front of the walk. In units of a CTA's 32 tokens, which take `tile` us when the SM is full; the least sum wins.
// us of the forward, with one segment and as chosen (bf16, D = 1536, N = 16 where nothing else is said):
//   1 x 65536 tokens 9263, 1529   1 x 4096 584, 127   4 x 2048 301, 208   8 x 2047, padded 452, 385   16 x 1024 305 (one is chosen)
//   2 x 1537, D = 384, float32 214, 47   2 x 4096, D = 1024, N = 64 548, 509
// and with its gradients: 8 x 1024 829, 672   2 x 1537, D = 384, float32 763, 134   2 x 1024, D = 1024, N = 64 540, 558 (one is better)
void sel_split(SelParams& p, bool back) {
    const int64_t ch = sel_channels(p.N), ctas = (int64_t)p.B * p.G * ((p.Dg + ch - 1) / ch), tiles = (p.L + kSelTile - 1) / kSelTile;
    if (ctas <= 0 || tiles <= 0) return;
    const double tile = back ? 8.5 : 3.3, first = back ? 0.2 : 0.4;
    auto full = [](int64_t n) { return std::max<double>(1.6, (double)((n + 147) / 148)); };
    double best = 1e30;
    for (int64_t g = 1; g <= 256 && (g == 1 || 4 * g <= tiles); ++g) {
        const int64_t per = (tiles + g - 1) / g;
        if ((tiles + per - 1) / per != g) continue;  // (the same split with fewer segments)
        double t = (double)per * full(ctas * g) * tile;
        if (g > 1) t += (double)per * full(ctas * (g - 1)) * tile * first + 4.0 + 0.15 * (double)g;
        if (t < best) best = t, p.nseg = (int)g, p.seg_tokens = (int)(per * kSelTile);
    }
}

size_t np_of(const SelParams& p) { return 4 * (size_t)sel_lanes(p.N); }
size_t kept_bytes(const SelParams& p) { return align_up((size_t)p.B * ((p.L + kSelKeep - 1) / kSelKeep) * p.D * np_of(p) * 4); }
struct SegBytes {
    size_t h, dt, copy;
    size_t all() const { return h + dt + copy; }
};
SegBytes seg_bytes(const SelParams& p) {
    if (p.nseg == 1) return {0, 0, 0};
    const size_t n = (size_t)p.nseg * p.B * p.D;
    return {align_up(n * np_of(p) * 4), align_up(n * 4), p.S_in && p.S_in == p.S_out ? align_up((size_t)p.B * p.D * p.N * 4) : 0};
}
// The walk back leaves each CTA's part of dB and dC, 8 (4 lanes)^2 / 1024 bytes a token and channel: at N <= 16 half of a float32
// [B, L, D], at N > 64 32 times it. Beyond 1 GiB and one such tensor the walk goes in ranges of tokens
// (bf16 training steps, N = 128, all tokens at once and as cut: 1 x 16384 x 1536 18.4, 18.3 ms; 16 x 1024 x 1536 15.9, 15.0; 8 x 2048 x 2048
// 21.0, 21.1).
size_t bc_row_bytes(const SelParams& p) {  // of one token of all sequences
    const size_t ch = sel_channels(p.N), blocks = (p.Dg + ch - 1) / ch;
    return blocks * p.B * p.G * 2 * np_of(p) * 4;
}
int sel_ranges(const SelParams& p) { return (p.seg_tokens + p.range_tokens - 1) / p.range_tokens; }
void sel_cut_ranges(SelParams& p) {
    p.range_tokens = p.seg_tokens;
    p.rows = p.L;
    const size_t most = std::max((size_t)1 << 30, (size_t)p.B * p.L * p.D * 4), tile = bc_row_bytes(p) * p.nseg * kSelTile;
    if (tile == 0 || (size_t)p.L <= most / bc_row_bytes(p)) return;
    const int64_t tiles = p.seg_tokens / kSelTile, held = std::max<int64_t>(1, (int64_t)(most / tile)), ranges = (tiles + held - 1) / held;
    if (ranges <= 1) return;
    p.range_tokens = (int)((tiles + ranges - 1) / ranges * kSelTile);
    p.rows = p.nseg * p.range_tokens;
}
struct SelBwdBytes {
    SegBytes fwd, rev;
    size_t kept, bc, a, d, carry;
    size_t all() const { return std::max(fwd.all(), rev.all()) + kept + bc + a + d + carry; }
};
SelBwdBytes sel_bwd_bytes(const SelParams& fwd, const SelParams& rev, bool handover) {
    const size_t parts = (size_t)rev.B * rev.nseg, states = align_up(parts * rev.D * np_of(rev) * 4);
    return {handover ? SegBytes{0, 0, 0} : seg_bytes(fwd), seg_bytes(rev), handover ? 0 : kept_bytes(rev), align_up(bc_row_bytes(rev) * rev.rows), states,
            align_up(parts * 2 * rev.D * 4), sel_ranges(rev) > 1 ? states : 0};
}

int fill_sel_fwd(const subq_selective_fwd_args* a, SelParams& p, bool& step) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    int rc = check_sel(a->desc, p);
    if (rc) return rc;
    const int t = a->desc.dtype;
    const bool need = p.B > 0 && p.L > 0 && p.D > 0;
    if ((rc = tensor3(a->u, "u", t, need, p.u)) || (rc = tensor3(a->dt, "dt", t, need, p.dt)) || (rc = tensor3(a->z, "z", t, false, p.z)) ||
        (rc = tensor3(a->B, "B", t, need, p.Bm)) || (rc = tensor3(a->C, "C", t, need, p.C)) || (rc = tensor3(a->out, "out", t, need, p.out)) ||
        (rc = aligned(a->state_in, 4, "state_in")) || (rc = aligned(a->state_out, 4, "state_out")))
        return rc;
    p.S_in = a->state_in;
    p.S_out = a->state_out;
    if (a->handover && reinterpret_cast<uintptr_t>(a->handover) % kAlign != 0) return fail(SUBQ_ERR_WORKSPACE, "handover must be 256-byte aligned");
    p.kept = static_cast<float*>(a->handover);
    step = p.L <= kSelStepTokens && !p.kept;
    if (!step) sel_split(p, false);
    return SUBQ_OK;
}

int check_sel_fwd_apart(const SelParams& p, int t) {
    const int64_t state = (int64_t)p.B * p.D * p.N * 4, one = (int64_t)p.D * 4;
    return check_apart({of_rows("out", p.out, p.B, p.L, 1, p.D, t), of_bytes("state_out", p.S_out, state), of_bytes("handover", p.kept, (int64_t)kept_bytes(p))},
                       {of_rows("u", p.u, p.B, p.L, 1, p.D, t), of_rows("dt", p.dt, p.B, p.L, 1, p.D, t), of_rows("z", p.z, p.B, p.L, 1, p.D, t),
                        of_rows("B", p.Bm, p.B, p.L, p.G, p.N, t), of_rows("C", p.C, p.B, p.L, p.G, p.N, t), of_mask(p.mask, p.mask_sb, p.B, p.L),
                        of_bytes("state_in", p.S_in == p.S_out ? nullptr : p.S_in, state), of_bytes("A", p.A, one * p.N), of_bytes("D", p.Dw, one),
                        of_bytes("dt_bias", p.dt_bias, one)});
}

void take_segments(SelParams& p, const SegBytes& n, unsigned char* at) {
    p.seg_h = reinterpret_cast<float*>(at);
    p.seg_dt = reinterpret_cast<float*>(at + n.h);
}

// The walk over all tokens, with its segments' launch before it where there are any.
cudaError_t run_sel_fwd(SelParams& p, int dtype, const SegBytes& n, unsigned char* ws, cudaStream_t st, int* launches) {
    cudaError_t err = cudaSuccess;
    *launches = 1;
    if (p.nseg > 1) {
        take_segments(p, n, ws);
        if (n.copy) {  // the last segment writes the state that the others still read
            float* copy = reinterpret_cast<float*>(ws + n.h + n.dt);
            err = cudaMemcpyAsync(copy, p.S_in, (size_t)p.B * p.D * p.N * 4, cudaMemcpyDeviceToDevice, st);
            p.S_in = copy;
        }
        if (err == cudaSuccess) err = launch_sel_fwd(p, dtype, kSelSegments, st);
        *launches = 2;
    }
    return err == cudaSuccess ? launch_sel_fwd(p, dtype, kSelWalk, st) : err;
}

int fill_sel_bwd(const subq_selective_bwd_args* a, SelParams& fwd, SelParams& rev) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    SelParams p;
    int rc = check_sel(a->desc, p);
    if (rc) return rc;
    const int t = a->desc.dtype;
    const bool need = p.B > 0 && p.L > 0 && p.D > 0;
    SelTensor dB, dC;
    if ((rc = tensor3(a->u, "u", t, need, p.u)) || (rc = tensor3(a->dt, "dt", t, need, p.dt)) || (rc = tensor3(a->z, "z", t, false, p.z)) ||
        (rc = tensor3(a->B, "B", t, need, p.Bm)) || (rc = tensor3(a->C, "C", t, need, p.C)) || (rc = tensor3(a->dout, "dout", t, need, p.dout)) ||
        (rc = tensor3(a->du, "du", t, need, p.du)) || (rc = tensor3(a->ddt, "ddt", t, need, p.ddt)) || (rc = tensor3(a->dz, "dz", t, need && a->z.data, p.dz)) ||
        (rc = tensor3(a->dB, "dB", t, need, dB)) || (rc = tensor3(a->dC, "dC", t, need, dC)) || (rc = aligned(a->state_in, 4, "state_in")) ||
        (rc = aligned(a->dstate_out, 4, "dstate_out")) || (rc = aligned(a->dstate_in, 4, "dstate_in")) || (rc = aligned(a->dA, 4, "dA")) ||
        (rc = aligned(a->dD, 4, "dD")) || (rc = aligned(a->ddt_bias, 4, "ddt_bias")))
        return rc;
    if (!a->z.data) p.dz = SelTensor{};
    if (p.D > 0 && !a->dA) return fail(SUBQ_ERR_INVALID_ARGUMENT, "dA is null");
    p.dB = const_cast<void*>(dB.p); p.dB_sb = dB.sb; p.dB_sl = dB.sl; p.dB_sg = dB.sg;
    p.dC = const_cast<void*>(dC.p); p.dC_sb = dC.sb; p.dC_sl = dC.sl; p.dC_sg = dC.sg;
    p.S_in = a->state_in;
    p.dS_out = a->dstate_out;
    p.dS_in = a->dstate_in;
    p.dA = a->dA;
    p.dD = a->dD;
    p.dbias = a->ddt_bias;
    if (a->handover && reinterpret_cast<uintptr_t>(a->handover) % kAlign != 0) return fail(SUBQ_ERR_WORKSPACE, "handover must be 256-byte aligned");
    p.kept = static_cast<float*>(const_cast<void*>(a->handover));
    fwd = rev = p;
    sel_split(fwd, false);
    // (one CTA reads the gradient that another one's result would overwrite)
    if (!(p.dS_in && p.dS_in == p.dS_out)) sel_split(rev, true);
    sel_cut_ranges(rev);
    const int64_t state = (int64_t)p.B * p.D * p.N * 4, one = (int64_t)p.D * 4;
    return check_apart({of_rows("du", p.du, p.B, p.L, 1, p.D, t), of_rows("ddt", p.ddt, p.B, p.L, 1, p.D, t), of_rows("dz", p.dz, p.B, p.L, 1, p.D, t),
                        of_rows("dB", dB, p.B, p.L, p.G, p.N, t), of_rows("dC", dC, p.B, p.L, p.G, p.N, t), of_bytes("dstate_in", p.dS_in, state),
                        of_bytes("dA", p.dA, one * p.N), of_bytes("dD", p.dD, one), of_bytes("ddt_bias", p.dbias, one)},
                       {of_rows("u", p.u, p.B, p.L, 1, p.D, t), of_rows("dt", p.dt, p.B, p.L, 1, p.D, t), of_rows("z", p.z, p.B, p.L, 1, p.D, t),
                        of_rows("B", p.Bm, p.B, p.L, p.G, p.N, t), of_rows("C", p.C, p.B, p.L, p.G, p.N, t), of_rows("dout", p.dout, p.B, p.L, 1, p.D, t),
                        of_mask(p.mask, p.mask_sb, p.B, p.L), of_bytes("state_in", p.S_in, state),
                        of_bytes("dstate_out", p.dS_out == p.dS_in ? nullptr : p.dS_out, state), of_bytes("A", p.A, one * p.N), of_bytes("D", p.Dw, one),
                        of_bytes("dt_bias", p.dt_bias, one), of_bytes("handover", p.kept, (int64_t)kept_bytes(p))});
}

// -------------------------------------------------------------- convolution
int fill_conv(const subq_causal_conv_args* a, ConvParams& p, bool bwd) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    if (a->batch < 0 || a->seq_len < 0 || a->channels < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative batch, seq_len or channels");
    if (a->width < 2 || a->width > 4) return fail(SUBQ_ERR_UNSUPPORTED, "the convolution's width must be 2, 3 or 4");
    if (a->batch > 65535 || a->seq_len > (int64_t)1 << 30 || a->channels > (int64_t)1 << 24)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "batch above 65535, seq_len above 2^30 or channels above 2^24");
    if (!known_type(a->dtype)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "the convolution supports float32, float16 and bfloat16");
    if (a->silu != 0 && a->silu != 1) return fail(SUBQ_ERR_INVALID_ARGUMENT, "silu must be 0 or 1");
    if (a->mask && a->mask_stride_b < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "mask has a negative stride");
    p = ConvParams{};
    p.B = (int)a->batch; p.L = (int)a->seq_len; p.D = (int)a->channels; p.W = (int)a->width;
    p.silu = a->silu;
    p.w = a->weight; p.bias = a->bias;
    p.mask = a->mask;
    p.mask_sb = a->mask ? a->mask_stride_b : 0;
    p.S_in = a->state_in;
    const int t = a->dtype;
    const size_t es = elem_size(t);
    const bool need = p.B > 0 && p.L > 0 && p.D > 0;
    int rc;
    if ((rc = tensor3(a->x, "x", t, need, p.x)) || (rc = aligned(a->weight, 4, "weight")) || (rc = aligned(a->bias, 4, "bias")) ||
        (rc = aligned(a->state_in, es, "state_in")))
        return rc;
    if (p.D > 0 && !p.w) return fail(SUBQ_ERR_INVALID_ARGUMENT, "weight is null");
    // (a CTA has 32 channels, or pieces of them, and 8 runs of 8 tokens)
    if (((int64_t)p.B * ((p.L + 7) / 8) + 7) / 8 * ((p.D + 31) / 32) > 0x7fffffff) return fail(SUBQ_ERR_UNSUPPORTED, "batch * seq_len * channels is too large for one call");
    const int64_t window = (int64_t)p.B * (p.W - 1) * p.D * (int64_t)es, one = (int64_t)p.D * 4;
    if (!bwd) {
        p.S_out = a->state_out;
        if ((rc = tensor3(a->y, "y", t, need, p.y)) || (rc = aligned(a->state_out, es, "state_out"))) return rc;
        return check_apart({of_rows("y", p.y, p.B, p.L, 1, p.D, t), of_bytes("state_out", p.S_out, window)},
                           {of_rows("x", p.x, p.B, p.L, 1, p.D, t), of_mask(p.mask, p.mask_sb, p.B, p.L), of_bytes("weight", p.w, one * p.W), of_bytes("bias", p.bias, one),
                            of_bytes("state_in", p.S_in == p.S_out ? nullptr : p.S_in, window)});
    }
    p.dS_out = a->dstate_out;
    p.dS_in = a->dstate_in;
    p.dw = a->dweight;
    p.db = a->dbias;
    if ((rc = tensor3(a->dy, "dy", t, need, p.dy)) || (rc = tensor3(a->dx, "dx", t, need, p.dx)) || (rc = aligned(a->dstate_out, es, "dstate_out")) ||
        (rc = aligned(a->dstate_in, es, "dstate_in")) || (rc = aligned(a->dweight, 4, "dweight")) || (rc = aligned(a->dbias, 4, "dbias")))
        return rc;
    if (p.D > 0 && !p.dw) return fail(SUBQ_ERR_INVALID_ARGUMENT, "dweight is null");
    if (need) conv_bwd_split(p);
    return check_apart({of_rows("dx", p.dx, p.B, p.L, 1, p.D, t), of_bytes("dstate_in", p.dS_in, window), of_bytes("dweight", p.dw, one * p.W), of_bytes("dbias", p.db, one)},
                       {of_rows("x", p.x, p.B, p.L, 1, p.D, t), of_rows("dy", p.dy, p.B, p.L, 1, p.D, t), of_mask(p.mask, p.mask_sb, p.B, p.L),
                        of_bytes("weight", p.w, one * p.W), of_bytes("bias", p.bias, one), of_bytes("state_in", p.S_in, window), of_bytes("dstate_out", p.dS_out, window)});
}
size_t conv_bwd_bytes(const ConvParams& p) {
    if (p.B == 0 || p.L == 0 || p.D == 0) return 0;
    return align_up(((size_t)p.parts * (p.W + 1) * p.D + (size_t)p.B) * 4);
}

// -------------------------------------------------------------- norm
int fill_rms(const subq_rms_norm_args* a, RmsNormParams& p, bool bwd) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    if (a->rows < 0 || a->dim <= 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative rows or dim <= 0");
    if (a->dim > kRmsMaxD) return fail(SUBQ_ERR_UNSUPPORTED, "dim above 16384 is not supported");
    const int x = a->x_dtype, r = a->r_dtype, y = a->y_dtype;
    if (!known_type(x) || !known_type(r)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "the norm supports float32, float16 and bfloat16");
    if (r != x && r != SUBQ_FP32) return fail(SUBQ_ERR_UNSUPPORTED, "the residual must have x's type or be float32");
    if (!bwd && y != x && y != SUBQ_E4M3 && !(x == SUBQ_FP32 && known_type(y)))
        return fail(SUBQ_ERR_UNSUPPORTED, "y must have x's type, be e4m3, or be 16 bits wide where x is float32");
    if (!(a->eps >= 0.f) || a->eps > 1e30f) return fail(SUBQ_ERR_INVALID_ARGUMENT, "eps must be >= 0 and finite");
    if (a->norm != 0 && a->norm != 1) return fail(SUBQ_ERR_INVALID_ARGUMENT, "norm must be 0 or 1");
    const bool some = a->rows > 0;
    const size_t ex = elem_size(x), er = elem_size(r);
    auto check = [&](const void* q, int64_t stride, size_t es, const char* name, bool need) {
        if (some && need && !q) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
        if (int rc = aligned(q, es, name)) return rc;
        if (q && stride < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
        return (int)SUBQ_OK;
    };
    auto rows = [&](const char* name, const void* at, int64_t stride, size_t es, int64_t width) -> Memory {
        return {name, {reinterpret_cast<uintptr_t>(at), (int64_t)(width * es), {a->rows, 1, 1}, {(__int128)stride * es, 0, 0}}};
    };
    p = RmsNormParams{};
    p.rows = a->rows; p.D = (int)a->dim; p.eps = a->eps; p.norm = a->norm; p.w = a->weight;
    p.r = a->r; p.r_s = a->r_stride;
    int rc = aligned(a->weight, 4, "weight");
    if (rc) return rc;
    if (!bwd) {
        const size_t ey = y == SUBQ_E4M3 ? 1 : elem_size(y);
        const int64_t blocks = (a->dim + 127) / 128;
        if ((rc = check(a->x, a->x_stride, ex, "x", true)) || (rc = check(a->residual, a->residual_stride, er, "residual", false)) ||
            (rc = check(a->r, a->r_stride, er, "r", false)) || (rc = check(a->y, a->y_stride, ey, "y", true)) ||
            (rc = check(a->scale, a->scale_stride, 4, "scale", y == SUBQ_E4M3)))
            return rc;
        p.x = a->x; p.x_s = a->x_stride;
        p.res = a->residual; p.res_s = a->residual_stride;
        p.y = a->y; p.y_s = a->y_stride;
        p.scale = a->scale; p.scale_s = a->scale_stride;
        // r may stand in x's or the residual's place, of one type and row stride: a row is read before it is written
        const bool on_x = p.r && p.r == p.x && ex == er && x == r && (p.r_s == p.x_s || p.rows == 1);
        const bool on_res = p.r && p.r == p.res && (p.r_s == p.res_s || p.rows == 1);
        return check_apart({rows("r", p.r, p.r_s, er, p.D), rows("y", p.y, p.y_s, ey, p.D), rows("scale", y == SUBQ_E4M3 ? p.scale : nullptr, p.scale_s, 4, blocks)},
                           {rows("x", on_x ? nullptr : p.x, p.x_s, ex, p.D), rows("residual", on_res ? nullptr : p.res, p.res_s, er, p.D), of_bytes("weight", p.w, (int64_t)p.D * 4)});
    }
    if ((rc = check(a->r, a->r_stride, er, "r", true)) || (rc = check(a->dy, a->dy_stride, ex, "dy", true)) || (rc = check(a->dr_next, a->dr_next_stride, er, "dr_next", false)) ||
        (rc = check(a->dx, a->dx_stride, ex, "dx", false)) || (rc = check(a->dres, a->dres_stride, er, "dres", false)) || (rc = aligned(a->dweight, 4, "dweight")))
        return rc;
    p.dy = a->dy; p.dy_s = a->dy_stride;
    p.dr = a->dr_next; p.dr_s = a->dr_next_stride;
    p.dx = a->dx; p.dx_s = a->dx_stride;
    p.dres = a->dres; p.dres_s = a->dres_stride;
    p.dw = a->dweight;
    return check_apart({rows("dx", p.dx, p.dx_s, ex, p.D), rows("dres", p.dres, p.dres_s, er, p.D), of_bytes("dweight", p.dw, (int64_t)p.D * 4)},
                       {rows("r", p.r, p.r_s, er, p.D), rows("dy", p.dy, p.dy_s, ex, p.D), rows("dr_next", p.dr, p.dr_s, er, p.D), of_bytes("weight", p.w, (int64_t)p.D * 4)});
}
size_t rms_bwd_bytes(const RmsNormParams& p) { return p.dw && p.rows > 0 ? align_up((size_t)kRmsParts * p.D * 4) : 0; }

cudaError_t clear(std::initializer_list<std::pair<float*, size_t>> all, cudaStream_t st) {
    for (const auto& x : all)
        if (x.first && x.second)
            if (cudaError_t err = cudaMemsetAsync(x.first, 0, x.second * 4, st)) return err;
    return cudaSuccess;
}

}  // namespace

extern "C" {

size_t subq_selective_scan_handover_bytes(const subq_selective_desc* d) {
    SelParams p;
    if (!d || check_sel(*d, p) != SUBQ_OK) return 0;
    return kept_bytes(p);
}

size_t subq_selective_scan_fwd_workspace_bytes(const subq_selective_fwd_args* a) {
    SelParams p;
    bool step;
    if (fill_sel_fwd(a, p, step) != SUBQ_OK || step) return 0;
    return seg_bytes(p).all();
}

size_t subq_selective_scan_bwd_workspace_bytes(const subq_selective_bwd_args* a) {
    SelParams fwd, rev;
    if (fill_sel_bwd(a, fwd, rev) != SUBQ_OK || rev.B == 0 || rev.L == 0 || rev.D == 0) return 0;
    return sel_bwd_bytes(fwd, rev, a->handover != nullptr).all();
}

int subq_selective_scan_fwd(const subq_selective_fwd_args* a) {
    SelParams p;
    bool step;
    int rc = fill_sel_fwd(a, p, step), launches = 0;
    if (rc || (rc = check_sel_fwd_apart(p, a->desc.dtype))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (p.B > 0 && p.D > 0 && (p.L > 0 || p.S_out)) {
        cudaError_t err;
        if (step || p.L == 0) {
            err = launch_sel_step(p, a->desc.dtype, st);
            launches = 1;
        } else {
            const SegBytes n = seg_bytes(p);
            if ((rc = check_workspace(a->workspace, a->workspace_bytes, n.all()))) return rc;
            err = run_sel_fwd(p, a->desc.dtype, n, static_cast<unsigned char*>(a->workspace), st, &launches);
        }
        if (err != cudaSuccess) return fail_cuda(err, "subq_selective_scan_fwd launch");
    }
    set_launches(launches);
    return SUBQ_OK;
}

int subq_selective_scan_bwd(const subq_selective_bwd_args* a) {
    SelParams fwd, p;
    int rc = fill_sel_bwd(a, fwd, p), launches = 0;
    if (rc) return rc;
    const int dt = a->desc.dtype;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    cudaError_t err = cudaSuccess;
    if (p.B == 0 || p.L == 0 || p.D == 0) {  // no token: the state's gradient passes through
        const size_t n = (size_t)p.B * p.D * p.N;
        err = clear({{p.dA, (size_t)p.D * p.N}, {p.dD, (size_t)p.D}, {p.dbias, (size_t)p.D}, {p.dS_out ? nullptr : p.dS_in, n}}, st);
        if (err == cudaSuccess && p.dS_in && p.dS_out && p.dS_in != p.dS_out && n) err = cudaMemcpyAsync(p.dS_in, p.dS_out, n * 4, cudaMemcpyDeviceToDevice, st);
        if (err != cudaSuccess) return fail_cuda(err, "subq_selective_scan_bwd");
        set_launches(0);
        return SUBQ_OK;
    }
    const SelBwdBytes n = sel_bwd_bytes(fwd, p, a->handover != nullptr);
    if ((rc = check_workspace(a->workspace, a->workspace_bytes, n.all()))) return rc;
    unsigned char* ws = static_cast<unsigned char*>(a->workspace);
    p.part_bc = reinterpret_cast<float*>(ws);
    p.part_a = reinterpret_cast<float*>(ws + n.bc);
    p.part_d = reinterpret_cast<float*>(ws + n.bc + n.a);
    if (n.carry) p.carry = reinterpret_cast<float*>(ws + n.bc + n.a + n.d + n.kept);
    unsigned char* segs = ws + n.bc + n.a + n.d + n.kept + n.carry;
    if (!a->handover) {
        fwd.kept = p.kept = reinterpret_cast<float*>(ws + n.bc + n.a + n.d);
        fwd.out = SelTensor{};  // the states alone
        err = run_sel_fwd(fwd, dt, n.fwd, segs, st, &launches);
    }
    if (err == cudaSuccess && p.nseg > 1) {
        take_segments(p, n.rev, segs);
        err = launch_sel_bwd(p, dt, kSelSegments, st);
        ++launches;
    }
    const int ranges = sel_ranges(p);
    for (int r = ranges - 1; r >= 0 && err == cudaSuccess; --r) {
        p.range0 = r * p.range_tokens;
        err = launch_sel_bwd(p, dt, kSelWalk, st);
        if (err == cudaSuccess) err = launch_sel_sums(p, dt, r == 0, st);
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_selective_scan_bwd launch");
    set_launches(launches + 2 * ranges + 1);
    return SUBQ_OK;
}

int subq_causal_conv_fwd(const subq_causal_conv_args* a) {
    ConvParams p;
    int rc = fill_conv(a, p, false), launches = 0;
    if (rc) return rc;
    if (p.B > 0 && p.D > 0 && (p.L > 0 || p.S_out)) {
        cudaError_t err = launch_conv_fwd(p, a->dtype, static_cast<cudaStream_t>(a->stream), &launches);
        if (err != cudaSuccess) return fail_cuda(err, "subq_causal_conv_fwd launch");
    }
    set_launches(launches);
    return SUBQ_OK;
}

size_t subq_causal_conv_bwd_workspace_bytes(const subq_causal_conv_args* a) {
    ConvParams p;
    return fill_conv(a, p, true) == SUBQ_OK ? conv_bwd_bytes(p) : 0;
}

int subq_causal_conv_bwd(const subq_causal_conv_args* a) {
    ConvParams p;
    int rc = fill_conv(a, p, true), launches = 0;
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    cudaError_t err;
    if (p.B == 0 || p.L == 0 || p.D == 0) {
        const size_t n = (size_t)p.B * (p.W - 1) * p.D * elem_size(a->dtype);
        err = clear({{p.dw, (size_t)p.D * p.W}, {p.db, (size_t)p.D}}, st);
        if (err == cudaSuccess && p.dS_in && n) err = p.dS_out ? cudaMemcpyAsync(p.dS_in, p.dS_out, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(p.dS_in, 0, n, st);
    } else {
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, conv_bwd_bytes(p)))) return rc;
        p.part = static_cast<float*>(a->workspace);
        err = launch_conv_bwd(p, a->dtype, st, &launches);
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_causal_conv_bwd launch");
    set_launches(launches);
    return SUBQ_OK;
}

int subq_rms_norm_fwd(const subq_rms_norm_args* a) {
    RmsNormParams p;
    int rc = fill_rms(a, p, false);
    if (rc) return rc;
    if (p.rows > 0) {
        cudaError_t err = launch_rms_norm(p, a->x_dtype, a->r_dtype, a->y_dtype == SUBQ_E4M3 ? -1 : a->y_dtype, static_cast<cudaStream_t>(a->stream));
        if (err != cudaSuccess) return fail_cuda(err, "subq_rms_norm_fwd launch");
    }
    set_launches(p.rows > 0);
    return SUBQ_OK;
}

size_t subq_rms_norm_bwd_workspace_bytes(const subq_rms_norm_args* a) {
    RmsNormParams p;
    return fill_rms(a, p, true) == SUBQ_OK ? rms_bwd_bytes(p) : 0;
}

int subq_rms_norm_bwd(const subq_rms_norm_args* a) {
    RmsNormParams p;
    int rc = fill_rms(a, p, true), launches = 0;
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    cudaError_t err;
    if (p.rows == 0) {
        err = clear({{p.dw, (size_t)p.D}}, st);
    } else {
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, rms_bwd_bytes(p)))) return rc;
        p.part = p.dw ? static_cast<float*>(a->workspace) : nullptr;
        err = launch_rms_norm_bwd(p, a->x_dtype, a->r_dtype, st, &launches);
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_rms_norm_bwd launch");
    set_launches(launches);
    return SUBQ_OK;
}

int subq_scaled_matmul(const subq_scaled_matmul_args* a) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    if (a->M < 0 || a->N < 0 || a->K < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative M, N or K");
    if (a->M > (int64_t)1 << 30 || a->N > (int64_t)1 << 24 || a->K > (int64_t)1 << 24)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "M above 2^30, N or K above 2^24");
    if (!known_type(a->out_dtype)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "the product's type must be float32, float16 or bfloat16");
    const int64_t nk = (a->K + 127) / 128, nb = (a->N + 127) / 128;
    const bool some = a->M > 0 && a->N > 0;
    const size_t es = elem_size(a->out_dtype);
    int rc;
    auto operand = [&](const void* q, int64_t stride, const char* name) {
        if (some && a->K > 0 && !q) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
        if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || stride % 16 != 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string("rows of ") + name + " must start on 16-byte boundaries");
        if (stride < a->K || stride >= (int64_t)1 << 40) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string("rows of ") + name + " overlap, or are too far apart");
        return (int)SUBQ_OK;
    };
    auto scales = [&](const void* q, int64_t stride, const char* name) {
        if (some && a->K > 0 && !q) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
        if (int bad = aligned(q, 4, name)) return bad;
        return stride < 0 ? fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride") : (int)SUBQ_OK;
    };
    if ((rc = operand(a->a, a->a_stride, "a")) || (rc = operand(a->b, a->b_stride, "b")) || (rc = scales(a->a_scale, a->a_scale_stride, "a_scale")) ||
        (rc = scales(a->b_scale, a->b_scale_stride, "b_scale")) || (rc = aligned(a->bias, 4, "bias")) || (rc = aligned(a->out, es, "out")))
        return rc;
    if (some && !a->out) return fail(SUBQ_ERR_INVALID_ARGUMENT, "out is null");
    if (a->out_stride < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "out has a negative stride");
    if ((a->M + 127) / 128 * ((a->N + 31) / 32) > 0x7fffffff) return fail(SUBQ_ERR_UNSUPPORTED, "M * N is too large for one call");
    if (a->K == 0 && a->M > 4 * 65535) return fail(SUBQ_ERR_UNSUPPORTED, "M is too large for a product without columns");
    auto rows = [&](const char* name, const void* at, int64_t n, int64_t stride, int64_t size, int64_t width) -> Memory {
        return {name, {reinterpret_cast<uintptr_t>(at), width * size, {n, 1, 1}, {(__int128)stride * size, 0, 0}}};
    };
    if ((rc = check_apart({rows("out", a->out, a->M, a->out_stride, (int64_t)es, a->N)},
                          {rows("a", a->a, a->M, a->a_stride, 1, a->K), rows("b", a->b, a->N, a->b_stride, 1, a->K), rows("a_scale", a->a_scale, a->M, a->a_scale_stride, 4, nk),
                           rows("b_scale", a->b_scale, nb, a->b_scale_stride, 4, nk), of_bytes("bias", a->bias, a->N * 4)})))
        return rc;
    if (some) {
        MatmulParams p{};
        p.M = a->M; p.N = (int)a->N; p.K = (int)a->K; p.nk = (int)nk;
        p.a = a->a; p.a_s = a->a_stride; p.b = a->b; p.b_s = a->b_stride;
        p.a_scale = a->a_scale; p.as_s = a->a_scale_stride; p.b_scale = a->b_scale; p.bs_s = a->b_scale_stride;
        p.bias = a->bias; p.out = a->out; p.out_s = a->out_stride;
        cudaError_t err = launch_scaled_matmul(p, a->out_dtype, static_cast<cudaStream_t>(a->stream));
        if (err != cudaSuccess) return fail_cuda(err, "subq_scaled_matmul launch");
    }
    set_launches(some);
    return SUBQ_OK;
}

}  // extern "C"
