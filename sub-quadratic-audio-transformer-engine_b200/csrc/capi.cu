// The C ABI (include/kernels.hpp): argument validation, workspace sizing,
// kernel-path selection and launch. No exception crosses this boundary.
#include <cuda_runtime.h>
#include <stdio.h>
#include <string.h>

#include <initializer_list>
#include <mutex>
#include <string>
#include <tuple>

#include "delta_common.cuh"
#include "delta_launch.h"
#include "kernels.hpp"
#include "overlap.h"
#include "scan_common.cuh"
#include "scan_launch.h"

namespace {

thread_local std::string g_last_error;
thread_local int g_last_path = SUBQ_PATH_AUTO;
thread_local int g_last_launches = 0;

int fail(int code, const std::string& msg) {
    g_last_error = msg;
    return code;
}

int fail_cuda(cudaError_t err, const char* where) {
    return fail(SUBQ_ERR_CUDA, std::string(where) + ": " + cudaGetErrorString(err));
}

size_t elem_size(int dtype) { return dtype == SUBQ_FP64 ? 8 : dtype == SUBQ_FP32 ? 4 : 2; }

constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// Common checks of a scan description; fills the scalar part of ScanParams.
int check_desc(const subq_scan_desc& d, subq::ScanParams& p) {
    if (d.batch < 0 || d.heads < 0 || d.seq_len < 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative batch, heads or seq_len");
    if (d.head_dim <= 0 || d.value_dim <= 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "head_dim and value_dim must be positive");
    if (d.batch > 65535 || d.heads > 65535 || d.seq_len > (int64_t)1 << 30)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "batch/heads above 65535 or seq_len above 2^30");
    if (d.head_dim > 256 || d.value_dim > 256)
        return fail(SUBQ_ERR_UNSUPPORTED, "head_dim and value_dim above 256 are not supported");
    if (d.dtype != SUBQ_FP32 && d.dtype != SUBQ_FP16 && d.dtype != SUBQ_BF16 && d.dtype != SUBQ_FP64)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "unknown dtype");
    if (d.decay_mode < SUBQ_DECAY_NONE || d.decay_mode > SUBQ_DECAY_PER_TOKEN)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "unknown decay_mode");
    if ((d.decay_mode == SUBQ_DECAY_PER_HEAD || d.decay_mode == SUBQ_DECAY_PER_TOKEN) && !d.log_gamma)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "log_gamma pointer required by decay_mode");
    if (d.path < SUBQ_PATH_AUTO || d.path > SUBQ_PATH_CHUNKED)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "unknown kernel path");
    if (!(d.clamp_min >= 0.f))
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "clamp_min must be >= 0");
    if (d.kv_heads < 0 || (d.kv_heads > 0 && d.heads % d.kv_heads != 0))
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "kv_heads must be 0 or a divisor of heads");
    if (d.reverse != 0 && d.reverse != 1) return fail(SUBQ_ERR_INVALID_ARGUMENT, "reverse must be 0 or 1");
    memset(&p, 0, sizeof(p));
    p.B = (int)d.batch; p.H = (int)d.heads; p.N = (int)d.seq_len;
    p.d = (int)d.head_dim; p.e = (int)d.value_dim;
    p.normalize = d.normalize ? 1 : 0;
    p.scale = d.scale;
    p.clamp_min = d.clamp_min;
    p.decay_mode = d.decay_mode;
    p.lg_scalar = d.log_gamma_scalar;
    p.log_gamma = d.log_gamma;
    p.mask = d.mask;
    p.mask_sb = d.mask ? d.mask_stride_b : 0;
    p.flush = d.flush_subnormal ? 1 : 0;
    p.kvg = (d.kv_heads > 0 && d.heads > 0) ? (int)(d.heads / d.kv_heads) : 1;
    p.reverse = d.reverse;
    return SUBQ_OK;
}

// `empty`: the call touches no element (B, H or N is 0), so a null pointer is fine.
int check_tensor(const subq_tensor4& t, const char* name, int dtype, bool empty) {
    if (!t.data && !empty) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    if (reinterpret_cast<uintptr_t>(t.data) % elem_size(dtype) != 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is not aligned to its element size");
    if (t.stride_b < 0 || t.stride_h < 0 || t.stride_n < 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
    return SUBQ_OK;
}

// Calls of at most this many tokens (streaming decode steps) run on the
// token-recurrent kernel under SUBQ_PATH_AUTO: a single-token step takes
// about 3.7 us there against about 13 us for one chunk of the tensor-core
// kernel (measured on B200 at B*H <= 48, CUDA-graph replay); the two meet
// near 16 tokens.
constexpr int kRecurrentMaxTokens = 16;

bool use_tc(const subq::ScanParams& p, int dtype, int path) {
    if (path == SUBQ_PATH_EXACT || path == SUBQ_PATH_CHUNKED || dtype == SUBQ_FP64) return false;
    if (path == SUBQ_PATH_AUTO && p.N <= kRecurrentMaxTokens) return false;
    return subq::tc_supported(p, dtype);
}

bool use_tc_bwd(const subq::ScanParams& p, int dtype, int path) {
    return use_tc(p, dtype, path) && subq::tc_bwd_supported(p, dtype);
}

// The automatic path takes the chunked forward while its workspace (about
// 0.8 KB per token-head at d = 64, 2.3 KB at d = 256) stays within this; larger
// calls run on the exact path, which needs none.
constexpr size_t kChunkMaxWorkspace = (size_t)4 << 30;

// The forward's kernel family when the tensor cores do not take the call.
int fwd_simt_path(const subq::ScanParams& p, int dtype, int path) {
    if (path == SUBQ_PATH_CHUNKED) return subq::chunk_fwd_usable(p, dtype) ? SUBQ_PATH_CHUNKED : -1;
    if (path == SUBQ_PATH_AUTO && p.N >= subq::kChunkMinTokens && subq::chunk_fwd_usable(p, dtype) &&
        subq::chunk_fwd_workspace_bytes(p) <= kChunkMaxWorkspace)
        return SUBQ_PATH_CHUNKED;
    return SUBQ_PATH_EXACT;
}

int fill_fwd(const subq_fwd_args* a, subq::ScanParams& p) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    int rc = check_desc(a->desc, p);
    if (rc) return rc;
    const int dt = a->desc.dtype;
    const bool empty = p.B == 0 || p.H == 0 || p.N == 0;
    if ((rc = check_tensor(a->q, "q", dt, empty)) || (rc = check_tensor(a->k, "k", dt, empty)) ||
        (rc = check_tensor(a->v, "v", dt, empty)) || (rc = check_tensor(a->o, "o", dt, empty)))
        return rc;
    p.q = a->q.data; p.q_sb = a->q.stride_b; p.q_sh = a->q.stride_h; p.q_sn = a->q.stride_n;
    p.k = a->k.data; p.k_sb = a->k.stride_b; p.k_sh = a->k.stride_h; p.k_sn = a->k.stride_n;
    p.v = a->v.data; p.v_sb = a->v.stride_b; p.v_sh = a->v.stride_h; p.v_sn = a->v.stride_n;
    p.o = a->o.data; p.o_sb = a->o.stride_b; p.o_sh = a->o.stride_h; p.o_sn = a->o.stride_n;
    p.S_in = a->state_in; p.z_in = a->norm_in;
    p.S_out = a->state_out; p.z_out = a->norm_out;
    p.seg_out = a->segment_states;
    return SUBQ_OK;
}

int fill_bwd(const subq_bwd_args* a, subq::ScanParams& p) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    int rc = check_desc(a->desc, p);
    if (rc) return rc;
    const int dt = a->desc.dtype;
    const bool empty = p.B == 0 || p.H == 0 || p.N == 0;
    if ((rc = check_tensor(a->q, "q", dt, empty)) || (rc = check_tensor(a->k, "k", dt, empty)) ||
        (rc = check_tensor(a->v, "v", dt, empty)) || (rc = check_tensor(a->dout, "dout", dt, empty)) ||
        (rc = check_tensor(a->dq, "dq", dt, empty)) || (rc = check_tensor(a->dk, "dk", dt, empty)) ||
        (rc = check_tensor(a->dv, "dv", dt, empty)))
        return rc;
    if (empty) return SUBQ_OK;
    const void* ins[] = {a->q.data, a->k.data, a->v.data, a->dout.data};
    const void* outs[] = {a->dq.data, a->dk.data, a->dv.data};
    for (const void* in : ins)
        for (const void* out : outs)
            if (in == out)
                return fail(SUBQ_ERR_ALIAS,
                            "subquadratic_attention_backward: gradient outputs must not alias inputs");
    if (a->dq.data == a->dk.data || a->dq.data == a->dv.data || a->dk.data == a->dv.data)
        return fail(SUBQ_ERR_ALIAS, "gradient outputs must be distinct buffers");
    p.q = a->q.data; p.q_sb = a->q.stride_b; p.q_sh = a->q.stride_h; p.q_sn = a->q.stride_n;
    p.k = a->k.data; p.k_sb = a->k.stride_b; p.k_sh = a->k.stride_h; p.k_sn = a->k.stride_n;
    p.v = a->v.data; p.v_sb = a->v.stride_b; p.v_sh = a->v.stride_h; p.v_sn = a->v.stride_n;
    p.g = a->dout.data; p.g_sb = a->dout.stride_b; p.g_sh = a->dout.stride_h; p.g_sn = a->dout.stride_n;
    p.o = a->dq.data; p.o_sb = a->dq.stride_b; p.o_sh = a->dq.stride_h; p.o_sn = a->dq.stride_n;
    p.dk = a->dk.data; p.dk_sb = a->dk.stride_b; p.dk_sh = a->dk.stride_h; p.dk_sn = a->dk.stride_n;
    p.dv = a->dv.data; p.dv_sb = a->dv.stride_b; p.dv_sh = a->dv.stride_h; p.dv_sn = a->dv.stride_n;
    p.S_in = a->state_in; p.z_in = a->norm_in;
    p.dlg = a->dlog_gamma;
    p.seg_in = a->segment_states;
    if (a->out.data) {
        if ((rc = check_tensor(a->out, "out", dt, false))) return rc;
        p.fo = a->out.data; p.fo_sb = a->out.stride_b; p.fo_sh = a->out.stride_h; p.fo_sn = a->out.stride_n;
    }
    return SUBQ_OK;
}

size_t exact_bwd_ws(const subq::ScanParams& p, int dtype) {
    return align_up(elem_size(dtype == SUBQ_FP64 ? SUBQ_FP64 : SUBQ_FP32) * 3 * (size_t)p.B * p.H * (size_t)p.N);
}

// Grouped K/V: the scan kernels write dk [B, H, N, d] and dv [B, H, N, e] per
// query head into contiguous buffers after the kernels' own workspace; group
// sums then write the caller's [B, kv_heads, N, *] gradients.
size_t gqa_dk_bytes(const subq::ScanParams& p, int dtype) {
    return align_up(elem_size(dtype) * (size_t)p.B * p.H * (size_t)p.N * (size_t)p.d);
}
size_t gqa_bytes(const subq::ScanParams& p, int dtype) {
    if (p.kvg <= 1) return 0;
    return gqa_dk_bytes(p, dtype) + align_up(elem_size(dtype) * (size_t)p.B * p.H * (size_t)p.N * (size_t)p.e);
}

size_t scan_bwd_ws(const subq::ScanParams& p, int dtype, bool tc) {
    if (!tc) return exact_bwd_ws(p, dtype);
    return subq::bwd1_usable(p) ? subq::bwd1_workspace_bytes(p) : subq::tc_bwd_workspace_bytes(p);
}

int check_workspace(void* ws, size_t have, size_t need) {
    if (need == 0) return SUBQ_OK;
    if (!ws) return fail(SUBQ_ERR_WORKSPACE, "workspace required: " + std::to_string(need) + " bytes");
    if (have < need)
        return fail(SUBQ_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) +
                                            " bytes, got " + std::to_string(have));
    if (reinterpret_cast<uintptr_t>(ws) % kAlign != 0)
        return fail(SUBQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    return SUBQ_OK;
}

}  // namespace

extern "C" {

int subq_abi_version(void) { return SUBQ_ABI_VERSION; }

const char* subq_last_error(void) { return g_last_error.c_str(); }

int subq_last_path(void) { return g_last_path; }

int subq_device_status(void* stream, int* status) {
    if (!status) return fail(SUBQ_ERR_INVALID_ARGUMENT, "status is null");
    int v = 0;
    cudaError_t err = subq::tc_read_status(static_cast<cudaStream_t>(stream), &v);
    if (err != cudaSuccess) return fail_cuda(err, "subq_device_status");
    *status = v;
    return SUBQ_OK;
}

int subq_last_launches(void) { return g_last_launches; }

int subq_selftest_wait_timeout(int polls, void* stream) {
    if (polls < 1 || polls > (1 << 20)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "polls must be in [1, 2^20]");
    cudaError_t err = subq::tc_selftest_wait_timeout(polls, static_cast<cudaStream_t>(stream));
    if (err != cudaSuccess) return fail_cuda(err, "subq_selftest_wait_timeout launch");
    g_last_launches = 1;
    return SUBQ_OK;
}

size_t subq_fwd_workspace_bytes(const subq_fwd_args* a) {
    subq::ScanParams p;
    if (fill_fwd(a, p) != SUBQ_OK) return 0;
    if (use_tc(p, a->desc.dtype, a->desc.path)) return subq::tc_fwd_workspace_bytes(p);
    if (fwd_simt_path(p, a->desc.dtype, a->desc.path) == SUBQ_PATH_CHUNKED) return subq::chunk_fwd_workspace_bytes(p);
    return 0;
}

size_t subq_segment_states_bytes(const subq_fwd_args* a) {
    subq::ScanParams p;
    if (fill_fwd(a, p) != SUBQ_OK || p.B == 0 || p.H == 0) return 0;
    return use_tc(p, a->desc.dtype, a->desc.path) ? subq::tc_segment_states_bytes(p) : 0;
}

size_t subq_bwd_workspace_bytes(const subq_bwd_args* a) {
    subq::ScanParams p;
    if (fill_bwd(a, p) != SUBQ_OK) return 0;
    return scan_bwd_ws(p, a->desc.dtype, use_tc_bwd(p, a->desc.dtype, a->desc.path)) + gqa_bytes(p, a->desc.dtype);
}

int subq_fwd(const subq_fwd_args* a) {
    subq::ScanParams p;
    int rc = fill_fwd(a, p);
    if (rc) return rc;
    const bool tc = use_tc(p, a->desc.dtype, a->desc.path);
    if (a->desc.path == SUBQ_PATH_TENSORCORE && !tc)
        return fail(SUBQ_ERR_UNSUPPORTED, "tensor-core path needs bf16/fp16 with head_dim = value_dim = 64");
    const int simt = tc ? SUBQ_PATH_TENSORCORE : fwd_simt_path(p, a->desc.dtype, a->desc.path);
    if (simt < 0)
        return fail(SUBQ_ERR_UNSUPPORTED,
                    "chunked path needs fp32/fp16/bf16, head_dim <= 256, forward time and no decay fallback");
    const int used = tc ? SUBQ_PATH_TENSORCORE : simt;
    if (p.B == 0 || p.H == 0) {
        g_last_path = used;
        g_last_launches = 0;
        return SUBQ_OK;
    }
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    cudaError_t err;
    int launches = 0;
    if (p.seg_out) {  // "not written" until the tensor-core kernel stamps its segment count
        err = cudaMemsetAsync(p.seg_out, 0, 256, st);
        if (err != cudaSuccess) return fail_cuda(err, "subq_fwd segment_states header");
        if (!tc) p.seg_out = nullptr;
    }
    if (tc) {
        const size_t need = subq::tc_fwd_workspace_bytes(p);
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, need))) return rc;
        p.ws = static_cast<float*>(a->workspace);
        err = subq::launch_fwd_tc(p, a->desc.dtype, st, &launches);
    } else if (used == SUBQ_PATH_CHUNKED) {
        const size_t need = subq::chunk_fwd_workspace_bytes(p);
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, need))) return rc;
        p.ws = static_cast<float*>(a->workspace);
        err = subq::launch_fwd_chunk(p, a->desc.dtype, st, &launches);
    } else {
        err = subq::launch_fwd_exact(p, a->desc.dtype, st);
        launches = 1;
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_fwd launch");
    g_last_path = used;
    g_last_launches = launches;
    return SUBQ_OK;
}

int subq_bwd(const subq_bwd_args* a) {
    subq::ScanParams p;
    int rc = fill_bwd(a, p);
    if (rc) return rc;
    const bool tc = use_tc_bwd(p, a->desc.dtype, a->desc.path);
    if (a->desc.path == SUBQ_PATH_TENSORCORE && !tc)
        return fail(SUBQ_ERR_UNSUPPORTED, "tensor-core path needs bf16/fp16 with head_dim = value_dim = 64");
    if (!tc && subq::exact_bwd_smem_bytes(p.d, p.e, p.normalize, a->desc.dtype == SUBQ_FP64 ? 8 : 4) > 220 * 1024)
        return fail(SUBQ_ERR_UNSUPPORTED, "backward state d x (e+1) does not fit in shared memory");
    if (p.B == 0 || p.H == 0 || p.N == 0) {
        g_last_path = tc ? SUBQ_PATH_TENSORCORE : SUBQ_PATH_EXACT;
        g_last_launches = 0;
        return SUBQ_OK;
    }
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    cudaError_t err;
    int launches = 0;
    const size_t scan_need = scan_bwd_ws(p, a->desc.dtype, tc);
    const size_t need = scan_need + gqa_bytes(p, a->desc.dtype);
    if ((rc = check_workspace(a->workspace, a->workspace_bytes, need))) return rc;
    p.ws = static_cast<float*>(a->workspace);
    if (p.kvg > 1) {  // per-query-head dk, dv into the workspace; summed per group below
        char* base = static_cast<char*>(a->workspace) + scan_need;
        p.dk = base;
        p.dk_sn = p.d, p.dk_sh = (int64_t)p.N * p.d, p.dk_sb = p.dk_sh * p.H;
        p.dv = base + gqa_dk_bytes(p, a->desc.dtype);
        p.dv_sn = p.e, p.dv_sh = (int64_t)p.N * p.e, p.dv_sb = p.dv_sh * p.H;
    }
    if (tc && subq::bwd1_usable(p)) {  // one pass from the forward's handover
        err = subq::launch_bwd1(p, a->desc.dtype, st, &launches);
    } else if (tc) {
        err = subq::launch_bwd_tc(p, a->desc.dtype, st, &launches);
    } else {
        err = subq::launch_bwd_exact(p, a->desc.dtype, st);
        launches = 1;
    }
    if (err == cudaSuccess && p.kvg > 1) {
        const int Hkv = p.H / p.kvg;
        err = subq::launch_group_sum(p.dk, a->dk.data, a->desc.dtype, p.B, Hkv, p.kvg, p.N, p.d, a->dk.stride_b,
                                     a->dk.stride_h, a->dk.stride_n, st);
        if (err == cudaSuccess)
            err = subq::launch_group_sum(p.dv, a->dv.data, a->desc.dtype, p.B, Hkv, p.kvg, p.N, p.e, a->dv.stride_b,
                                         a->dv.stride_h, a->dv.stride_n, st);
        launches += 2;
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_bwd launch");
    g_last_path = tc ? SUBQ_PATH_TENSORCORE : SUBQ_PATH_EXACT;
    g_last_launches = launches;
    return SUBQ_OK;
}

int subq_feature_map(void* x, int64_t n, int32_t dtype, void* stream) {
    if (n < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative element count");
    if (n > 0 && !x) return fail(SUBQ_ERR_INVALID_ARGUMENT, "x is null");
    if (dtype != SUBQ_FP32 && dtype != SUBQ_FP16 && dtype != SUBQ_BF16)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "subq_feature_map supports float32, float16 and bfloat16");
    cudaError_t err = subq::launch_feature_map(x, n, dtype, static_cast<cudaStream_t>(stream));
    if (err != cudaSuccess) return fail_cuda(err, "subq_feature_map launch");
    g_last_launches = n > 0 ? 1 : 0;
    return SUBQ_OK;
}

// Checks of a per-head RMSNorm call; fills p. Rows must be 16-byte aligned
// (the kernels move 8 elements per thread).
static int fill_rms(const subq_rmsnorm_args* a, subq::RmsParams& p, bool bwd) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    if (a->batch < 0 || a->heads < 0 || a->seq_len < 0 || a->head_dim <= 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative batch, heads or seq_len, or head_dim <= 0");
    if (a->batch > 65535 || a->heads > 65535 || a->seq_len > (int64_t)1 << 30)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "batch/heads above 65535 or seq_len above 2^30");
    if (a->dtype != SUBQ_FP32 && a->dtype != SUBQ_FP16 && a->dtype != SUBQ_BF16)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "head RMSNorm supports float32, float16 and bfloat16");
    if (!subq::rms_supported_dim((int)a->head_dim))
        return fail(SUBQ_ERR_UNSUPPORTED, "head RMSNorm needs head_dim 8, 16, 32, 64, 128 or 256");
    if (!(a->eps >= 0.f) || a->eps > 1e30f) return fail(SUBQ_ERR_INVALID_ARGUMENT, "eps must be >= 0 and finite");
    p = subq::RmsParams{};
    p.B = (int)a->batch; p.H = (int)a->heads; p.N = (int)a->seq_len; p.D = (int)a->head_dim;
    p.eps = a->eps;
    p.w = a->weight;
    const bool empty = p.B == 0 || p.H == 0 || p.N == 0;
    const size_t es = elem_size(a->dtype);
    auto rows_aligned = [&](const subq_tensor4& t, const char* name) {
        int rc = check_tensor(t, name, a->dtype, empty);
        if (rc) return rc;
        if (reinterpret_cast<uintptr_t>(t.data) % 16 != 0 || (t.stride_b * es) % 16 != 0 ||
            (t.stride_h * es) % 16 != 0 || (t.stride_n * es) % 16 != 0)
            return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + ": rows must start on 16-byte boundaries");
        return (int)SUBQ_OK;
    };
    int rc = rows_aligned(a->x, "x");
    if (rc) return rc;
    p.x = a->x.data; p.x_sb = a->x.stride_b; p.x_sh = a->x.stride_h; p.x_sn = a->x.stride_n;
    if (!bwd) {
        if ((rc = rows_aligned(a->y, "y"))) return rc;
        p.y = a->y.data; p.y_sb = a->y.stride_b; p.y_sh = a->y.stride_h; p.y_sn = a->y.stride_n;
    } else {
        if ((rc = rows_aligned(a->dy, "dy")) || (rc = rows_aligned(a->dx, "dx"))) return rc;
        p.dy = a->dy.data; p.dy_sb = a->dy.stride_b; p.dy_sh = a->dy.stride_h; p.dy_sn = a->dy.stride_n;
        p.dx = a->dx.data; p.dx_sb = a->dx.stride_b; p.dx_sh = a->dx.stride_h; p.dx_sn = a->dx.stride_n;
        p.dw = a->dweight;
    }
    // dense (b, n, h) row order: row r at element r * D
    const int64_t D = p.D, H = p.H, N = p.N;
    auto dense = [&](const subq_tensor4& t) {
        return t.stride_h == D && t.stride_n == H * D && (t.stride_b == N * H * D || p.B == 1);
    };
    p.dense = (dense(a->x) ? 1 : 0) | (!bwd && dense(a->y) ? 2 : 0) | (bwd && dense(a->dy) ? 4 : 0) |
              (bwd && dense(a->dx) ? 8 : 0);
    return SUBQ_OK;
}

size_t subq_head_rmsnorm_bwd_workspace_bytes(const subq_rmsnorm_args* a) {
    subq::RmsParams p;
    if (fill_rms(a, p, true) != SUBQ_OK || !a->dweight) return 0;
    return align_up((size_t)subq::rms_blocks(p) * p.D * sizeof(float));
}

int subq_head_rmsnorm_fwd(const subq_rmsnorm_args* a) {
    subq::RmsParams p;
    int rc = fill_rms(a, p, false);
    if (rc) return rc;
    g_last_launches = 0;
    if (p.B == 0 || p.H == 0 || p.N == 0) return SUBQ_OK;
    cudaError_t err = subq::launch_rms_fwd(p, a->dtype, static_cast<cudaStream_t>(a->stream));
    if (err != cudaSuccess) return fail_cuda(err, "subq_head_rmsnorm_fwd launch");
    g_last_launches = 1;
    return SUBQ_OK;
}

int subq_head_rmsnorm_bwd(const subq_rmsnorm_args* a) {
    subq::RmsParams p;
    int rc = fill_rms(a, p, true);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    g_last_launches = 0;
    if (p.B == 0 || p.H == 0 || p.N == 0) {  // no rows: dweight is 0
        if (p.dw) {
            cudaError_t err = cudaMemsetAsync(p.dw, 0, sizeof(float) * p.D, st);
            if (err != cudaSuccess) return fail_cuda(err, "subq_head_rmsnorm_bwd dweight");
        }
        return SUBQ_OK;
    }
    if (p.dw) {
        const size_t need = (size_t)subq::rms_blocks(p) * p.D * sizeof(float);
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, need))) return rc;
        p.part = static_cast<float*>(a->workspace);
    }
    cudaError_t err = subq::launch_rms_bwd(p, a->dtype, st);
    if (err != cudaSuccess) return fail_cuda(err, "subq_head_rmsnorm_bwd launch");
    g_last_launches = p.dw ? 2 : 1;
    return SUBQ_OK;
}

// ------------------------------------------------------------ gated delta rule
namespace {

// Calls of at most this many tokens take the token-recurrent kernel (12 heads of 64 x 64: 13 us at 8 tokens, 19.5 at 16,
// 28 at 24 against 19.5 us for a chunk; 16 x 12 heads: 21.5 at 16 and 36 at 32 against 30; 256 x 12: 140 and 263 against 259).
constexpr int kDeltaRecurrentMaxTokens = 16;

int delta_gate(const subq_gate& g, const char* name, subq::DeltaGate& out) {
    if (reinterpret_cast<uintptr_t>(g.data) % 4 != 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is not aligned to its element size");
    if (g.data && (g.stride_b < 0 || g.stride_h < 0 || g.stride_n < 0))
        return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
    out = {g.data, g.stride_b, g.stride_h, g.stride_n};
    return SUBQ_OK;
}

int check_delta(const subq_delta_desc& d, subq::DeltaParams& p) {
    if (d.batch < 0 || d.heads < 0 || d.seq_len < 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative batch, heads or seq_len");
    if (d.head_dim <= 0 || d.value_dim <= 0)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "head_dim and value_dim must be positive");
    if (d.batch > 65535 || d.heads > 65535 || d.seq_len > (int64_t)1 << 30)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "batch/heads above 65535 or seq_len above 2^30");
    if (d.head_dim > 256 || d.value_dim > 256)
        return fail(SUBQ_ERR_UNSUPPORTED, "head_dim and value_dim above 256 are not supported");
    if (d.dtype != SUBQ_FP32 && d.dtype != SUBQ_FP16 && d.dtype != SUBQ_BF16)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "the gated delta rule supports float32, float16 and bfloat16");
    if (d.path != SUBQ_PATH_AUTO && d.path != SUBQ_PATH_EXACT && d.path != SUBQ_PATH_CHUNKED)
        return fail(SUBQ_ERR_INVALID_ARGUMENT, "the gated delta rule has the paths auto, exact and chunked");
    for (int64_t x : {d.q_heads, d.k_heads, d.v_heads})
        if (x < 0 || (x > 0 && d.heads % x != 0))
            return fail(SUBQ_ERR_INVALID_ARGUMENT, "q_heads, k_heads and v_heads must be 0 or divisors of heads");
    if (!(d.scale >= -3e38f && d.scale <= 3e38f)) return fail(SUBQ_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (d.mask && d.mask_stride_b < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "mask has a negative stride");
    p = subq::DeltaParams{};
    p.B = (int)d.batch; p.H = (int)d.heads; p.N = (int)d.seq_len; p.d = (int)d.head_dim; p.e = (int)d.value_dim;
    p.nc = (int)((d.seq_len + subq::kDeltaC - 1) / subq::kDeltaC);
    p.scale = d.scale;
    p.mask = d.mask;
    p.mask_sb = d.mask ? d.mask_stride_b : 0;
    int rc = delta_gate(d.beta, "beta", p.beta);
    if (rc) return rc;
    if ((rc = delta_gate(d.log_gamma, "log_gamma", p.lg))) return rc;
    // one CTA per (sequence, 64 tokens) and per (sequence, 32 value columns)
    const int64_t bh = d.batch * d.heads;
    if (bh * (p.nc > 8 ? p.nc : 8) > (int64_t)0x7fffffff)
        return fail(SUBQ_ERR_UNSUPPORTED, "batch * heads * seq_len is too large for one call");
    return SUBQ_OK;
}

int delta_tensor(const subq_tensor4& t, const char* name, const subq_delta_desc& d, int64_t heads, bool empty, subq::DeltaTensor& out) {
    int rc = check_tensor(t, name, d.dtype, empty);
    if (rc) return rc;
    const int64_t es = (int64_t)elem_size(d.dtype);
    out.p = t.data;
    out.sb = t.stride_b; out.sh = t.stride_h; out.sn = t.stride_n;
    out.group = heads > 0 && d.heads > 0 ? (int)(d.heads / heads) : 1;
    out.vec = reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && t.stride_b * es % 16 == 0 && t.stride_h * es % 16 == 0 &&
              t.stride_n * es % 16 == 0;
    return SUBQ_OK;
}

// Segments of a sequence that are walked side by side when there are few sequences. A walk over n chunks takes n steps, and
// about 3 more to begin and end, of a time that depends on the type and d (below) and not on the number of CTAs, up to one
// CTA per SM. With G segments a first pass finds the states: the first segment's own state, for the others their own state
// and what they do to the one before them, but for the last. Its steps take 0.7 of the walk's, or 1.1 where two CTAs share
// an SM. The walk itself then takes n / G steps, the join 1.4 us a segment (2 us above d = 64), and the two launches 8 us.
// G is the count with the least sum, taken where that is a tenth below the single walk's. Device time of a captured call,
// us, single and cut with the count that the rule takes (other counts were at most 2 % faster):
//   bf16, d = 64:  1 x 12 heads, 65536 tokens   2696, 1139 (G = 6)   2 x 12, 8192     381, 260 (G = 3)   1 x 4, 4096   174, 66 (G = 10)
//                  3 x 12 heads, 16384 tokens    795, 721 (G = 2)    4 x 12, 4096     227, none (G = 2: 291, more CTAs than SMs)
//                  1 x 1 head, 65536 tokens     2509, 201 (G = 38)   float16:  1 x 4, 4096   238, 82 (G = 10)
//   float32:       2 x 12 heads, 1537 tokens     150, 119 (G = 3)    1 x 4, 16384    1102, 231 (G = 18)
//   d = 128:       1 x 4 heads, 8192 tokens      481, 176 (bf16, G = 6)   1036, 303 (float16, G = 9)   1243, 430 (float32, G = 6)
//
// The walk back over the chunks is cut the same way. Its first pass has a whole step's work (the products with dO beside
// the chain, for the identity's columns too, where dO is 0), so the sum has to be a fifth below. The gradients' call from
// the forward's handover, us, single and cut:
//   bf16, d = 64:  1 x 12 heads, 65536 tokens   3809, 2194 (G = 4)   2 x 12, 8192     612, 490 (G = 3)   1 x 4, 4096   217, 90 (G = 10)
//                  3 x 12 heads, 16384 tokens   1415, none (G = 2: 1382)              4 x 12, 4096     432, none (G = 2: 516)
//                  1 x 1 head, 65536 tokens     2996, 289 (G = 38)   float16:  1 x 4, 4096   270, 119 (G = 10)
//   float32:       2 x 12 heads, 1537 tokens     238, none (G = 3: 229)                1 x 4, 16384   1231, 420 (G = 18)
//   d = 128:       1 x 4 heads, 8192 tokens      631, 342 (bf16, G = 6)   1395, 623 (float16, G = 6)   1620, 721 (float32, G = 6)
struct DeltaSplit {
    int nseg, chunks;
};
DeltaSplit delta_split(const subq::DeltaParams& p, int dtype, bool back = false) {
    const int64_t bh = (int64_t)p.B * p.H, ncb = (p.e + 31) / 32, ndb = (p.d + 31) / 32;
    const int wide = p.d > 64;
    constexpr double kSteps[3][2] = {{4.3, 9.2}, {3.6, 8.0}, {2.4, 3.7}};  // us: float32, float16, bfloat16
    const double step = kSteps[dtype == SUBQ_FP32 ? 0 : dtype == SUBQ_FP16 ? 1 : 2][wide], join = wide ? 2.0 : 1.4, launches = 8.0;
    const bool pairs = dtype == (wide ? SUBQ_FP16 : SUBQ_BF16);  // two CTAs of the first pass per SM (chain_ctas)
    auto waves = [](int64_t ctas, int64_t slots) { return (double)((ctas + slots - 1) / slots); };
    double best = (back ? 0.8 : 0.9) * (p.nc + 3) * step * waves(bh * ncb, 148);
    DeltaSplit s = {1, p.nc};
    if (back && p.dS_in && p.dS_in == p.dS_out) return s;  // (one CTA reads what another one's result would overwrite)
    for (int g = 2; g <= 64 && 2 * g <= p.nc; ++g) {
        const int chunks = (p.nc + g - 1) / g;
        if ((p.nc + chunks - 1) / chunks != g) continue;  // (the same split with fewer segments)
        const int64_t ctas = bh * ((g - 1) * (ncb + ndb) - ndb);
        const double states = back ? waves(ctas, 148) : !pairs || ctas <= 148 ? 0.7 * waves(ctas, 148) : 1.1 * waves(ctas, 296);
        const double t = (chunks + 3) * step * (waves(bh * g * ncb, 148) + states) + g * join + launches;
        if (t < best) best = t, s = {g, chunks};
    }
    return s;
}

struct DeltaBytes {
    size_t gates, Y, P, S0, W;  // the handover's parts
    size_t seg_S, seg_M, seg_in;  // workspace, where a sequence is cut into segments
    size_t segs() const { return seg_S + seg_M + seg_in; }
};
DeltaBytes delta_bytes(const subq::DeltaParams& p, int dtype) {
    const size_t nx = subq::kDeltaPlanes, chunks = (size_t)p.B * p.H * p.nc;
    const size_t ncw = 2 * ((p.e + subq::kDeltaCols - 1) / subq::kDeltaCols), dp = p.d <= 64 ? 64 : 128;
    const size_t mat = align_up(chunks * nx * subq::kYBlocks * 512);
    const int nseg = delta_split(p, dtype).nseg;
    const size_t slots = (size_t)p.B * p.H * (nseg - 1) * sizeof(float);
    const size_t copy = nseg > 1 && p.S_in && p.S_in == p.S_out ? (size_t)p.B * p.H * p.d * p.e * sizeof(float) : 0;
    return {align_up(chunks * sizeof(subq::DeltaGates)), mat, mat, align_up(chunks * ncw * (dp / 16) * nx * 512),
            align_up(chunks * ncw * 4 * nx * 512), align_up(slots * p.d * p.e), align_up(slots * dp * dp), align_up(copy)};
}

void delta_handover(subq::DeltaParams& p, const DeltaBytes& n, void* at) {
    p.gates = static_cast<subq::DeltaGates*>(at);
    p.Y = static_cast<unsigned char*>(at) + n.gates;
    p.P = p.Y + n.Y;
    p.S0 = p.P + n.P;
    p.W = p.S0 + n.S0;
}

void delta_segments(subq::DeltaParams& p, int dtype, const DeltaBytes& n, void* at) {
    const DeltaSplit s = delta_split(p, dtype);
    p.nseg = s.nseg;
    p.seg_chunks = s.chunks;
    p.seg_S = static_cast<float*>(at);
    p.seg_M = reinterpret_cast<float*>(static_cast<char*>(at) + n.seg_S);
    p.seg_in = n.seg_in ? reinterpret_cast<float*>(static_cast<char*>(at) + n.seg_S + n.seg_M) : nullptr;
}

struct Memory {
    const char* name;
    subq::MemRows rows;
};
Memory of_tensor(const char* name, const subq::DeltaTensor& t, const subq::DeltaParams& p, int width, int dtype) {
    const __int128 es = (__int128)elem_size(dtype);
    return {name, {reinterpret_cast<uintptr_t>(t.p), (int64_t)(width * es), {p.B, p.H / t.group, p.N}, {t.sb * es, t.sh * es, t.sn * es}}};
}
Memory of_gate(const char* name, const subq::DeltaGate& g, const subq::DeltaParams& p) {
    return {name, {reinterpret_cast<uintptr_t>(g.p), 4, {p.B, p.H, p.N}, {(__int128)4 * g.sb, (__int128)4 * g.sh, (__int128)4 * g.sn}}};
}
Memory of_bytes(const char* name, const void* at, int64_t bytes) { return {name, {reinterpret_cast<uintptr_t>(at), bytes}}; }
Memory of_mask(const subq::DeltaParams& p) {
    return {"mask", {reinterpret_cast<uintptr_t>(p.mask), p.N, {p.B, 1, 1}, {p.mask_sb, 0, 0}}};
}

// An output's rows must be apart, from one another and from every input's and other output's.
int check_apart(std::initializer_list<Memory> out_list, std::initializer_list<Memory> in_list) {
    const Memory *outs = out_list.begin(), *ins = in_list.begin();
    const int no = (int)out_list.size(), ni = (int)in_list.size();
    for (int i = 0; i < no; ++i) {
        if (subq::rows_overlap_themselves(outs[i].rows))
            return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string("rows of ") + outs[i].name + " overlap");
        for (int j = 0; j < ni + i; ++j) {
            const Memory& other = j < ni ? ins[j] : outs[j - ni];
            if (subq::rows_overlap(outs[i].rows, other.rows))
                return fail(SUBQ_ERR_ALIAS, std::string(outs[i].name) + " shares memory with " + other.name);
        }
    }
    return SUBQ_OK;
}

int check_delta_fwd_apart(const subq::DeltaParams& p, int dtype) {
    const int64_t state = (int64_t)p.B * p.H * p.d * p.e * 4;
    const std::initializer_list<Memory> outs = {of_tensor("o", p.o, p, p.e, dtype), of_bytes("state_out", p.S_out, state)};
    const std::initializer_list<Memory> ins = {of_tensor("q", p.q, p, p.d, dtype), of_tensor("k", p.k, p, p.d, dtype), of_tensor("v", p.v, p, p.e, dtype),
                          of_gate("beta", p.beta, p), of_gate("log_gamma", p.lg, p), of_mask(p),
                          of_bytes("state_in", p.S_in == p.S_out ? nullptr : p.S_in, state)};  // (in place is allowed)
    return check_apart(outs, ins);
}

int check_delta_bwd_apart(const subq::DeltaParams& p, int dtype) {
    const int64_t state = (int64_t)p.B * p.H * p.d * p.e * 4, gates = (int64_t)p.B * p.H * p.N * 4;
    const std::initializer_list<Memory> outs = {of_tensor("dq", p.dq, p, p.d, dtype), of_tensor("dk", p.dk, p, p.d, dtype), of_tensor("dv", p.dv, p, p.e, dtype),
                           of_bytes("dbeta", p.dbeta, gates), of_bytes("dlog_gamma", p.dlg, gates), of_bytes("dstate_in", p.dS_in, state)};
    const std::initializer_list<Memory> ins = {of_tensor("q", p.q, p, p.d, dtype), of_tensor("k", p.k, p, p.d, dtype), of_tensor("v", p.v, p, p.e, dtype),
                          of_tensor("dout", p.g, p, p.e, dtype), of_gate("beta", p.beta, p), of_gate("log_gamma", p.lg, p), of_mask(p),
                          of_bytes("state_in", p.S_in, state),
                          of_bytes("dstate_out", p.dS_out == p.dS_in ? nullptr : p.dS_out, state)};
    return check_apart(outs, ins);
}

int fill_delta_fwd(const subq_delta_fwd_args* a, subq::DeltaParams& p, int& path) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    const subq_delta_desc& d = a->desc;
    int rc = check_delta(d, p);
    if (rc) return rc;
    const bool empty = p.B == 0 || p.H == 0 || p.N == 0;
    if ((rc = delta_tensor(a->q, "q", d, d.q_heads, empty, p.q)) || (rc = delta_tensor(a->k, "k", d, d.k_heads, empty, p.k)) ||
        (rc = delta_tensor(a->v, "v", d, d.v_heads, empty, p.v)) || (rc = delta_tensor(a->o, "o", d, d.heads, empty, p.o)))
        return rc;
    for (const void* in : {a->q.data, a->k.data, a->v.data})
        if (!empty && a->o.data == in) return fail(SUBQ_ERR_ALIAS, "o must not be q, k or v");
    p.S_in = a->state_in;
    p.S_out = a->state_out;
    path = d.path;
    if (path == SUBQ_PATH_AUTO)
        path = p.d > 128 || (p.N <= kDeltaRecurrentMaxTokens && !a->handover) ? SUBQ_PATH_EXACT : SUBQ_PATH_CHUNKED;
    if (path == SUBQ_PATH_CHUNKED && p.d > 128)
        return fail(SUBQ_ERR_UNSUPPORTED, "the chunked path needs head_dim <= 128");
    if (path == SUBQ_PATH_EXACT && a->handover)
        return fail(SUBQ_ERR_UNSUPPORTED, "the handover is filled by the chunked path (head_dim <= 128) only");
    return SUBQ_OK;
}

int fill_delta_bwd(const subq_delta_bwd_args* a, subq::DeltaParams& p) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    const subq_delta_desc& d = a->desc;
    int rc = check_delta(d, p);
    if (rc) return rc;
    if (d.path == SUBQ_PATH_EXACT || p.d > 128)
        return fail(SUBQ_ERR_UNSUPPORTED, "the backward of the gated delta rule has the chunked path (head_dim <= 128) only");
    const bool empty = p.B == 0 || p.H == 0 || p.N == 0;
    if ((rc = delta_tensor(a->q, "q", d, d.q_heads, empty, p.q)) || (rc = delta_tensor(a->k, "k", d, d.k_heads, empty, p.k)) ||
        (rc = delta_tensor(a->v, "v", d, d.v_heads, empty, p.v)) || (rc = delta_tensor(a->dout, "dout", d, d.heads, empty, p.g)) ||
        (rc = delta_tensor(a->dq, "dq", d, d.q_heads, empty, p.dq)) ||
        (rc = delta_tensor(a->dk, "dk", d, d.k_heads, empty, p.dk)) ||
        (rc = delta_tensor(a->dv, "dv", d, d.v_heads, empty, p.dv)))
        return rc;
    if (!empty) {
        if (!a->dbeta) return fail(SUBQ_ERR_INVALID_ARGUMENT, "dbeta is null");
        const void* outs[] = {a->dq.data, a->dk.data, a->dv.data};
        for (const void* in : {a->q.data, a->k.data, a->v.data, a->dout.data})
            for (const void* out : outs)
                if (in == out) return fail(SUBQ_ERR_ALIAS, "gradient outputs must not alias inputs");
        if (outs[0] == outs[1] || outs[0] == outs[2] || outs[1] == outs[2])
            return fail(SUBQ_ERR_ALIAS, "gradient outputs must be distinct buffers");
    }
    p.S_in = a->state_in;
    p.dS_out = a->dstate_out;
    p.dS_in = a->dstate_in;
    p.dbeta = a->dbeta;
    p.dlg = a->dlog_gamma;
    return SUBQ_OK;
}

// Workspace of the backward: dS, Z, the walk back's segments, float32 gradients per state head of shared
// q, k, v, and the forward's part where no handover is given.
struct DeltaBwdBytes {
    DeltaBytes fwd;
    DeltaSplit rev;  // of the walk back
    size_t rev_S, rev_M, dq, dk, dv, total;
};
DeltaBwdBytes delta_bwd_bytes(const subq::DeltaParams& p, int dtype, bool handover) {
    DeltaBwdBytes n;
    n.fwd = delta_bytes(p, dtype);
    n.rev = delta_split(p, dtype, true);
    const size_t slots = (size_t)p.B * p.H * (n.rev.nseg - 1) * sizeof(float), dp = p.d <= 64 ? 64 : 128;
    n.rev_S = align_up(slots * p.d * p.e);
    n.rev_M = align_up(slots * dp * dp);
    const size_t tokens = (size_t)p.B * p.H * p.N;
    n.dq = p.q.group > 1 ? align_up(tokens * p.d * 4) : 0;
    n.dk = p.k.group > 1 ? align_up(tokens * p.d * 4) : 0;
    n.dv = p.v.group > 1 ? align_up(tokens * p.e * 4) : 0;
    n.total = n.fwd.S0 + n.fwd.W + n.rev_S + n.rev_M + n.dq + n.dk + n.dv + (handover ? 0 : n.fwd.gates + n.fwd.Y + n.fwd.P + n.fwd.S0 + n.fwd.W + n.fwd.segs());
    return n;
}

}  // namespace

size_t subq_delta_handover_bytes(const subq_delta_desc* d) {
    subq::DeltaParams p;
    if (!d || check_delta(*d, p) != SUBQ_OK || p.d > 128) return 0;
    const DeltaBytes n = delta_bytes(p, d->dtype);
    return n.gates + n.Y + n.P + n.S0 + n.W;
}

size_t subq_delta_fwd_workspace_bytes(const subq_delta_fwd_args* a) {
    subq::DeltaParams p;
    int path;
    if (fill_delta_fwd(a, p, path) != SUBQ_OK || path != SUBQ_PATH_CHUNKED) return 0;
    const DeltaBytes n = delta_bytes(p, a->desc.dtype);
    return n.segs() + (a->handover ? 0 : n.gates + n.Y + n.P);
}

size_t subq_delta_bwd_workspace_bytes(const subq_delta_bwd_args* a) {
    subq::DeltaParams p;
    if (fill_delta_bwd(a, p) != SUBQ_OK) return 0;
    return delta_bwd_bytes(p, a->desc.dtype, a->handover != nullptr).total;
}

int subq_delta_fwd(const subq_delta_fwd_args* a) {
    subq::DeltaParams p;
    int path, launches = 1;
    int rc = fill_delta_fwd(a, p, path);
    if (rc || (rc = check_delta_fwd_apart(p, a->desc.dtype))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    g_last_launches = 0;
    if (p.B == 0 || p.H == 0 || (p.N == 0 && !p.S_out)) {
        g_last_path = path;
        return SUBQ_OK;
    }
    cudaError_t err;
    if (path == SUBQ_PATH_EXACT || p.N == 0) {
        err = subq::launch_delta_step(p, a->desc.dtype, st);
    } else {
        const DeltaBytes n = delta_bytes(p, a->desc.dtype);
        const size_t segs = n.segs();
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, segs + (a->handover ? 0 : n.gates + n.Y + n.P)))) return rc;
        delta_segments(p, a->desc.dtype, n, a->workspace);
        if (a->handover) {
            if (reinterpret_cast<uintptr_t>(a->handover) % kAlign != 0)
                return fail(SUBQ_ERR_WORKSPACE, "handover must be 256-byte aligned");
            delta_handover(p, n, a->handover);
        } else {
            delta_handover(p, n, static_cast<char*>(a->workspace) + segs);
            p.S0 = p.W = nullptr;  // not kept
        }
        err = subq::launch_delta_fwd(p, a->desc.dtype, st);
        launches = p.nseg > 1 ? 4 : 2;
    }
    if (err != cudaSuccess) return fail_cuda(err, "subq_delta_fwd launch");
    g_last_path = path;
    g_last_launches = launches;
    return SUBQ_OK;
}

int subq_delta_bwd(const subq_delta_bwd_args* a) {
    subq::DeltaParams p;
    int rc = fill_delta_bwd(a, p);
    if (rc || (rc = check_delta_bwd_apart(p, a->desc.dtype))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    g_last_launches = 0;
    cudaError_t err = cudaSuccess;
    if (p.B == 0 || p.H == 0 || p.N == 0) {  // no token: the state's gradient passes through
        const size_t bytes = (size_t)p.B * p.H * p.d * p.e * sizeof(float);
        if (p.dS_in && bytes && p.dS_in != p.dS_out)
            err = p.dS_out ? cudaMemcpyAsync(p.dS_in, p.dS_out, bytes, cudaMemcpyDeviceToDevice, st)
                           : cudaMemsetAsync(p.dS_in, 0, bytes, st);
        g_last_path = SUBQ_PATH_CHUNKED;
        return err == cudaSuccess ? (int)SUBQ_OK : fail_cuda(err, "subq_delta_bwd state gradient");
    }
    const int dt = a->desc.dtype;
    const DeltaBwdBytes n = delta_bwd_bytes(p, dt, a->handover != nullptr);
    if ((rc = check_workspace(a->workspace, a->workspace_bytes, n.total))) return rc;
    unsigned char* at = static_cast<unsigned char*>(a->workspace);
    auto take = [&](size_t bytes) {
        unsigned char* x = at;
        at += bytes;
        return x;
    };
    p.dS = take(n.fwd.S0);
    p.Z = take(n.fwd.W);
    unsigned char* rev = take(n.rev_S + n.rev_M);
    if (n.dq) p.dq32 = reinterpret_cast<float*>(take(n.dq));
    if (n.dk) p.dk32 = reinterpret_cast<float*>(take(n.dk));
    if (n.dv) p.dv32 = reinterpret_cast<float*>(take(n.dv));
    int first = 0, launches = 0;
    if (a->handover) {
        if (reinterpret_cast<uintptr_t>(a->handover) % kAlign != 0)
            return fail(SUBQ_ERR_WORKSPACE, "handover must be 256-byte aligned");
        delta_handover(p, n.fwd, const_cast<void*>(a->handover));
    } else {
        delta_segments(p, dt, n.fwd, at);
        delta_handover(p, n.fwd, at + n.fwd.segs());
        err = subq::launch_delta_fwd(p, dt, st);  // (o is null: states and corrections only)
        first = p.nseg > 1 ? 4 : 2;
    }
    p.nseg = n.rev.nseg;
    p.seg_chunks = n.rev.chunks;
    p.seg_S = reinterpret_cast<float*>(rev);
    p.seg_M = reinterpret_cast<float*>(rev + n.rev_S);
    p.seg_in = nullptr;
    if (err == cudaSuccess) err = subq::launch_delta_bwd(p, dt, st, &launches);
    if (err != cudaSuccess) return fail_cuda(err, "subq_delta_bwd launch");
    g_last_path = SUBQ_PATH_CHUNKED;
    g_last_launches = first + launches;
    return SUBQ_OK;
}

// ------------------------------------------------------------------ layer norm
static int fill_ln(const subq_layer_norm_args* a, subq::LnParams& p, bool bwd) {
    if (!a) return fail(SUBQ_ERR_INVALID_ARGUMENT, "null argument block");
    if (a->rows < 0 || a->dim <= 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, "negative rows or dim <= 0");
    if (a->dim > (int64_t)1 << 24) return fail(SUBQ_ERR_UNSUPPORTED, "dim above 2^24 is not supported");
    for (int32_t t : {a->x_dtype, a->y_dtype})
        if (t != SUBQ_FP32 && t != SUBQ_FP16 && t != SUBQ_BF16)
            return fail(SUBQ_ERR_INVALID_ARGUMENT, "layer norm supports float32, float16 and bfloat16");
    if (a->x_dtype != a->y_dtype && a->x_dtype != SUBQ_FP32)
        return fail(SUBQ_ERR_UNSUPPORTED, "x and y must share one dtype, or x be float32");
    if (!(a->eps >= 0.f) || a->eps > 1e30f) return fail(SUBQ_ERR_INVALID_ARGUMENT, "eps must be >= 0 and finite");
    auto check = [&](const void* q, int64_t stride, int dtype, const char* name) {
        if (a->rows > 0 && !q) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
        if (reinterpret_cast<uintptr_t>(q) % elem_size(dtype) != 0)
            return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " is not aligned to its element size");
        if (stride < 0) return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
        return (int)SUBQ_OK;
    };
    p = subq::LnParams{};
    p.rows = a->rows; p.D = (int)a->dim; p.eps = a->eps; p.w = a->weight;
    int rc = check(a->x, a->x_stride, a->x_dtype, "x");
    if (rc) return rc;
    p.x = a->x; p.x_s = a->x_stride;
    // rows of an output that overlap would be written by several CTAs; an output that is an input has to have its layout
    auto check_out = [&](const void* out, int64_t stride, int dtype, std::initializer_list<std::tuple<const void*, int64_t, int>> ins) {
        if (a->rows > 1 && stride < a->dim) return fail(SUBQ_ERR_INVALID_ARGUMENT, "rows of an output overlap");
        for (const auto& [in, in_stride, in_dtype] : ins)
            if (a->rows > 0 && in == out && (in_stride != stride || in_dtype != dtype))
                return fail(SUBQ_ERR_ALIAS, "an output in an input's place needs its type and row stride");
        return (int)SUBQ_OK;
    };
    if (!bwd) {
        if ((rc = check(a->y, a->y_stride, a->y_dtype, "y"))) return rc;
        if ((rc = check_out(a->y, a->y_stride, a->y_dtype, {{a->x, a->x_stride, a->x_dtype}}))) return rc;
        p.y = a->y; p.y_s = a->y_stride;
        p.b = a->bias;
        return SUBQ_OK;
    }
    if ((rc = check(a->dy, a->dy_stride, a->y_dtype, "dy")) || (rc = check(a->dx, a->dx_stride, a->x_dtype, "dx"))) return rc;
    if ((rc = check_out(a->dx, a->dx_stride, a->x_dtype, {{a->x, a->x_stride, a->x_dtype}, {a->dy, a->dy_stride, a->y_dtype}}))) return rc;
    p.dy = a->dy; p.dy_s = a->dy_stride;
    p.dx = a->dx; p.dx_s = a->dx_stride;
    p.dw = a->dweight;
    p.db = a->dbias;
    return SUBQ_OK;
}

// (An output in an input's place, which fill_ln has seen to be laid out like it, is read before it is written.)
static int check_ln_apart(const subq_layer_norm_args* a, bool bwd) {
    auto rows = [&](const char* name, const void* at, int64_t stride, int dtype, const void* in_place = nullptr) -> Memory {
        const __int128 es = (__int128)elem_size(dtype);
        return {name, {reinterpret_cast<uintptr_t>(at == in_place ? nullptr : at), (int64_t)(a->dim * es), {a->rows, 1, 1}, {stride * es, 0, 0}}};
    };
    auto param = [&](const char* name, const void* at) { return of_bytes(name, at, a->dim * 4); };
    if (!bwd) {
        const std::initializer_list<Memory> outs = {rows("y", a->y, a->y_stride, a->y_dtype)};
        const std::initializer_list<Memory> ins = {rows("x", a->x, a->x_stride, a->x_dtype, a->y), param("weight", a->weight), param("bias", a->bias)};
        return check_apart(outs, ins);
    }
    const std::initializer_list<Memory> outs = {rows("dx", a->dx, a->dx_stride, a->x_dtype), param("dweight", a->dweight), param("dbias", a->dbias)};
    const std::initializer_list<Memory> ins = {rows("x", a->x, a->x_stride, a->x_dtype, a->dx), rows("dy", a->dy, a->dy_stride, a->y_dtype, a->dx),
                          param("weight", a->weight)};
    return check_apart(outs, ins);
}

size_t subq_layer_norm_bwd_workspace_bytes(const subq_layer_norm_args* a) {
    subq::LnParams p;
    if (fill_ln(a, p, true) != SUBQ_OK || (!p.dw && !p.db) || p.rows == 0) return 0;
    return align_up(subq::ln_bwd_workspace_floats(p.rows, p.D) * sizeof(float));
}

int subq_layer_norm_fwd(const subq_layer_norm_args* a) {
    subq::LnParams p;
    int rc = fill_ln(a, p, false), launches = 0;
    if (rc || (rc = check_ln_apart(a, false))) return rc;
    if (p.rows > 0) {
        cudaError_t err = subq::launch_layer_norm(p, a->x_dtype, a->y_dtype, false, static_cast<cudaStream_t>(a->stream), &launches);
        if (err != cudaSuccess) return fail_cuda(err, "subq_layer_norm_fwd launch");
    }
    g_last_launches = launches;
    return SUBQ_OK;
}

int subq_layer_norm_bwd(const subq_layer_norm_args* a) {
    subq::LnParams p;
    int rc = fill_ln(a, p, true), launches = 0;
    if (rc || (rc = check_ln_apart(a, true))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    if (p.rows == 0) {  // no rows: the sums are 0
        for (float* x : {p.dw, p.db}) {
            cudaError_t err = x ? cudaMemsetAsync(x, 0, sizeof(float) * p.D, st) : cudaSuccess;
            if (err != cudaSuccess) return fail_cuda(err, "subq_layer_norm_bwd dweight");
        }
        g_last_launches = 0;
        return SUBQ_OK;
    }
    if (p.D > 8192 && (a->dx == a->x || a->dx == a->dy))
        return fail(SUBQ_ERR_ALIAS, "dx must not be x or dy for dim above 8192 (rows are read more than once)");
    if (p.dw || p.db) {
        const size_t need = align_up(subq::ln_bwd_workspace_floats(p.rows, p.D) * sizeof(float));
        if ((rc = check_workspace(a->workspace, a->workspace_bytes, need))) return rc;
        p.part = static_cast<float*>(a->workspace);
        const int64_t most = subq::kLnPartials;
        p.stats = p.part + (size_t)2 * p.D * (p.rows < most ? p.rows : most);
    }
    cudaError_t err = subq::launch_layer_norm(p, a->x_dtype, a->y_dtype, true, st, &launches);
    if (err != cudaSuccess) return fail_cuda(err, "subq_layer_norm_bwd launch");
    g_last_launches = launches;
    return SUBQ_OK;
}

int subq_device_info(int device, char* arch, size_t arch_len, size_t* memory_bytes, int* bf16_supported) {
    cudaDeviceProp prop;
    cudaError_t err = cudaGetDeviceProperties(&prop, device);
    if (err != cudaSuccess) return fail_cuda(err, "cudaGetDeviceProperties");
    if (arch && arch_len) snprintf(arch, arch_len, "SM %d.%d", prop.major, prop.minor);
    if (memory_bytes) *memory_bytes = prop.totalGlobalMem;
    if (bf16_supported) *bf16_supported = prop.major >= 8 ? 1 : 0;
    return SUBQ_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Allocation-free backward (subq_bwd_noalloc).
//
// Some callers cannot hand the library any device memory for scratch: a
// real-time audio callback must not block on, or fail in, an allocator in the
// middle of a frame, and a host that owns a fixed device budget (a pool sized
// up front) may not grow it per call. For them the backward runs with a
// scratch buffer that is part of this library's static device memory, placed
// when the module loads, so the call itself allocates nothing.
//
//  * Capacity: kNoAllocScratchBytes = 8 MiB against subq_bwd_workspace_bytes:
//    1,048,576 token-heads (B x H x N) on the recomputing tensor-core path (8
//    bytes each), about 699,000 with per-token decay (12 bytes each plus a
//    flag per sequence) and on the float32 exact path (12 bytes each), about
//    349,000 on the float64 exact path (24 bytes each); the one-pass backward
//    (given the forward's handover) takes a fixed 16.6 KB per SM whatever the
//    length; grouped K/V adds dK and dV per query head. A larger call is
//    rejected with SUBQ_ERR_WORKSPACE before anything is launched.
//  * Nothing in the scratch has to start at zero when the call begins: every
//    call writes each per-token entry it later reads (the clamped normaliser
//    and the quotient coefficient, the exact path's per-token values, or the
//    one-pass backward's adjoint sums) before reading it, and the decayed
//    path clears its per-sequence fallback flags itself (a memset on the
//    call's stream, not an allocation).
//  * One buffer per device: calls that overlap in time on one device (two
//    streams, or host threads without ordering between them) race on it, so
//    such callers must serialise their calls.
//  * The first call on a device looks the buffer's address up with
//    cudaGetSymbolAddress while that device is current; make that first call
//    before capturing any stream of the device, so the lookup is not part of
//    a capture.
namespace {

constexpr size_t kNoAllocScratchBytes = size_t(8) << 20;
static __device__ __align__(256) unsigned char g_noalloc_scratch[kNoAllocScratchBytes];

constexpr int kNoAllocMaxDevices = 64;
std::mutex g_noalloc_mu;
void* g_noalloc_ptr[kNoAllocMaxDevices] = {};

// Address of this device's scratch; looked up once per device.
int noalloc_scratch(void** out) {
    int dev = -1;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return fail_cuda(err, "subq_bwd_noalloc: cudaGetDevice");
    if (dev < 0 || dev >= kNoAllocMaxDevices)
        return fail(SUBQ_ERR_UNSUPPORTED, "subq_bwd_noalloc: device index above 63");
    std::lock_guard<std::mutex> lock(g_noalloc_mu);
    if (!g_noalloc_ptr[dev]) {
        void* p = nullptr;
        err = cudaGetSymbolAddress(&p, g_noalloc_scratch);
        if (err != cudaSuccess) return fail_cuda(err, "subq_bwd_noalloc: cudaGetSymbolAddress");
        g_noalloc_ptr[dev] = p;
    }
    *out = g_noalloc_ptr[dev];
    return SUBQ_OK;
}

}  // namespace

extern "C" int subq_bwd_noalloc(const subq_bwd_args* args) {
    if (!args) return fail(SUBQ_ERR_INVALID_ARGUMENT, "args is null");
    const size_t need = subq_bwd_workspace_bytes(args);
    if (need > kNoAllocScratchBytes)
        return fail(SUBQ_ERR_WORKSPACE, "subq_bwd_noalloc: this call needs " + std::to_string(need) +
                                            " bytes of scratch, above the built-in " +
                                            std::to_string(kNoAllocScratchBytes) +
                                            " bytes (8 MiB); use subq_bwd with a caller workspace");
    void* scratch = nullptr;
    int rc = noalloc_scratch(&scratch);
    if (rc) return rc;
    subq_bwd_args a = *args;
    a.workspace = scratch;
    a.workspace_bytes = kNoAllocScratchBytes;
    return subq_bwd(&a);
}
