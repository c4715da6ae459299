/*
 * subq-b200 — C ABI of the causal ELU+1 linear-attention scan (sm_100a).
 *
 * This header is the drop-in boundary for the reference's kernel layer. Each
 * entry point replaces one reference interface (paths relative to the
 * reference tree):
 *
 *   subq_fwd            run_attention_forward(AttentionContext&)         include/attention.hpp:23-24
 *                       run_attention_forward_raw<T>(...) (declared only)  include/kernels.hpp:56-61
 *                       the torch chunked forward chunkwise_flash_linear_attention /
 *                       _single_direction_causal_scan                    python/subq_audio/autograd.py:292-438
 *   subq_bwd            subquadratic_attention_backward<T>,
 *                       run_attention_backward_raw<T>                    include/kernels.hpp:44-54
 *                       run_attention_backward_ex(...)                   include/attention.hpp:26-32
 *                       _single_direction_causal_backward                python/subq_audio/autograd.py:441-544
 *   subq_feature_map    run_feature_map(TensorDescriptor&)               include/attention.hpp:22
 *   subq_head_rmsnorm_fwd / _bwd
 *                       SubQLinearAttention's per-head nn.RMSNorm and the
 *                       transpose copy after it                          python/subq_audio/autograd.py:706-710,763-769
 *   subq_delta_fwd / _bwd, subq_layer_norm_fwd / _bwd:
 *                       no counterpart: the gated delta rule beside the scan,
 *                       and the norm before a layer
 *   subq_selective_scan_fwd / _bwd, subq_causal_conv_fwd / _bwd, subq_rms_norm_fwd /
 *   _bwd, subq_scaled_matmul:
 *                       no counterpart: a selective state space block's operators
 *   subq_*_workspace_bytes, subq_last_error, subq_abi_version, subq_device_info:
 *                       no single counterpart; they carry the reference's
 *                       scratch allocation (attention_backward.cpp:305-361 allocated
 *                       per call) and its exception text (bindings.cpp:227-231) across
 *                       a C boundary.
 *
 * Conventions
 *   - Every call is stream-ordered on `stream` (a cudaStream_t, NULL = legacy
 *     default stream) and returns a subq_status; nothing throws across the ABI.
 *     subq_last_error() returns the message of the calling thread's last
 *     failing call.
 *   - The library allocates no device memory. Scratch comes from the caller
 *     as `workspace` (query its size with the *_workspace_bytes functions;
 *     256-byte alignment required).
 *   - Tensors are [B, H, N, D] views with element strides for b, h and n; the
 *     innermost dimension must be contiguous. q, k, v, o (and the gradients)
 *     share one dtype. State tensors are always float32.
 *   - Math (per (b,h) sequence, t = 0..N-1, m_t = mask, 1 if no mask):
 *       gamma_t = exp(log_gamma_t) (1 on masked tokens and with SUBQ_DECAY_NONE)
 *       S_t = gamma_t S_{t-1} + (m_t phi(k_t)) (m_t v_t)^T,   z_t = gamma_t z_{t-1} + m_t phi(k_t)
 *       normalize = 0:  o_t = m_t (scale phi(q_t))^T S_t
 *       normalize = 1:  o_t = m_t (scale phi(q_t))^T S_t / max((scale phi(q_t))^T z_t, clamp_min)
 *     with phi(x) = ELU(x) + 1. The reference's C++ engine is normalize = 0,
 *     scale = 1, scalar decay, flush_subnormal = 1; its torch path is
 *     normalize = 1, scale = 1/sqrt(D), clamp_min = 1e-5.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SUBQ_ABI_VERSION 5

typedef enum subq_status {
    SUBQ_OK = 0,
    SUBQ_ERR_INVALID_ARGUMENT = 1, /* shapes, strides, null pointers, alignment  */
    SUBQ_ERR_ALIAS = 2,            /* gradient outputs alias inputs (reference attention_backward.cpp:51-56) */
    SUBQ_ERR_UNSUPPORTED = 3,      /* a shape/dtype combination no kernel covers  */
    SUBQ_ERR_CUDA = 4,             /* a CUDA runtime error (message has the text) */
    SUBQ_ERR_TIMEOUT = 5,          /* a bounded device-side wait gave up          */
    SUBQ_ERR_WORKSPACE = 6,        /* workspace missing, too small or misaligned  */
    SUBQ_ERR_STATE = 7             /* device status: a backward's segment_states was not
                                      filled by the forward of the same call          */
} subq_status;

/* Same order as the reference's PrecisionMode (include/tensor.hpp:14-18);
 * SUBQ_FP64 (float64 storage and accumulation, exact path only) is an
 * addition for float64 gradient checks. */
typedef enum subq_dtype { SUBQ_FP32 = 0, SUBQ_FP16 = 1, SUBQ_BF16 = 2, SUBQ_FP64 = 3 } subq_dtype;

typedef enum subq_decay_mode {
    SUBQ_DECAY_NONE = 0,      /* gamma == 1                                     */
    SUBQ_DECAY_SCALAR = 1,    /* log_gamma_scalar for every token               */
    SUBQ_DECAY_PER_HEAD = 2,  /* log_gamma[h], float32 [H]                      */
    SUBQ_DECAY_PER_TOKEN = 3  /* log_gamma[(b*H + h)*N + t], float32 [B,H,N]   */
} subq_decay_mode;

/* Which kernel family a call may use. AUTO picks the tensor-core path when
 * the shape allows it (bf16/fp16, d = e = 64; with per-token decay bf16
 * only); otherwise the chunk-parallel float32 forward for calls of at least
 * 64 tokens (d <= 256, forward time, scalar gamma <= 1, at most 4 GiB of
 * workspace), and the exact
 * float32 path for the rest. Calls of at most 16 tokens (streaming decode
 * steps) take the exact, token-recurrent path, which is faster there. The
 * backward has no chunked variant: CHUNKED runs it on the exact path. */
typedef enum subq_kernel_path {
    SUBQ_PATH_AUTO = 0,
    SUBQ_PATH_EXACT = 1,       /* SIMT float32 sequential scan, any d, e <= 256          */
    SUBQ_PATH_TENSORCORE = 2,  /* tcgen05 chunked scan, bf16/fp16, d = e = 64            */
    SUBQ_PATH_CHUNKED = 3      /* SIMT float32 chunk-parallel forward, d <= 256, no reverse */
} subq_kernel_path;

typedef struct subq_tensor4 {
    void* data;
    int64_t stride_b, stride_h, stride_n; /* element strides; d is contiguous */
} subq_tensor4;

typedef struct subq_scan_desc {
    int64_t batch, heads, seq_len, head_dim, value_dim;
    int32_t dtype;           /* subq_dtype of q, k, v, o and of the gradients */
    int32_t normalize;       /* 0: engine form, 1: normalised form            */
    float scale;             /* multiplies phi(q)                             */
    float clamp_min;         /* lower clamp of the denominator                */
    int32_t decay_mode;      /* subq_decay_mode                               */
    float log_gamma_scalar;  /* SUBQ_DECAY_SCALAR                             */
    const float* log_gamma;  /* SUBQ_DECAY_PER_HEAD / SUBQ_DECAY_PER_TOKEN    */
    const uint8_t* mask;     /* [B, N] (row stride mask_stride_b), nonzero = live; NULL = all live */
    int64_t mask_stride_b;
    int32_t flush_subnormal; /* flush |S| < FLT_MIN to 0 after every update   */
    int32_t path;            /* subq_kernel_path                              */
    /* Grouped K/V (GQA, python/subq_audio/autograd.py:746-748): 0 or `heads`
     * = one K/V head per query head; else a divisor of `heads`, and query
     * head h reads K/V head h / (heads / kv_heads). k, v (and dk, dv) then
     * have kv_heads heads; the backward's dk, dv sum over each group, as the
     * reference's repeat_interleave does under autograd. The state S, z and
     * log gamma stay per query head. */
    int64_t kv_heads;
    /* 1: reverse time - token t sees itself and the later tokens, with the
     * decay of tokens t..tau-1 between key tau and query t: the second
     * direction of the bidirectional scan (python/subq_audio/autograd.py:
     * 407-433, which runs it on time-flipped copies). The caller combines the
     * two directions. The state runs from the end of the sequence. */
    int32_t reverse;
} subq_scan_desc;

typedef struct subq_fwd_args {
    subq_scan_desc desc;
    subq_tensor4 q, k, v, o;
    const float* state_in;  /* S [B,H,d,e] float32, NULL = zeros                 */
    const float* norm_in;   /* z [B,H,d] float32, NULL = zeros (normalize = 1)   */
    float* state_out;       /* final S, may equal state_in, NULL = not wanted    */
    float* norm_out;        /* final z, may equal norm_in, NULL = not wanted     */
    void* workspace;
    size_t workspace_bytes;
    void* stream;           /* cudaStream_t */
    /* Optional (NULL = not wanted): receives the state at the start of each
     * segment of each sequence as the tensor-core forward computes it,
     * subq_segment_states_bytes(args) bytes. Passing the same buffer to the
     * backward of the same call spares it recomputing those states (the
     * reference's backward recomputes them, autograd.py:207-222). */
    float* segment_states;
} subq_fwd_args;

typedef struct subq_bwd_args {
    subq_scan_desc desc;
    subq_tensor4 q, k, v, dout; /* inputs of the forward and the upstream gradient */
    subq_tensor4 dq, dk, dv;    /* outputs; must not alias q, k, v or dout          */
    const float* state_in;      /* the forward's initial S (NULL = zeros)           */
    const float* norm_in;       /* the forward's initial z (NULL = zeros)           */
    float* dlog_gamma;          /* [B,H,N] float32 d loss / d log(gamma_t), or NULL */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
    /* Optional: the segment_states buffer the forward of the same inputs
     * filled. Alone, it is used when it matches this call's segment split and
     * ignored otherwise. */
    const float* segment_states;
    /* Optional (ABI 4): the forward's output o of the same call. Given with
     * segment_states on the tensor-core path without decay, the backward runs
     * in one pass from what that forward handed over (its per-chunk states and
     * normalisers) instead of recomputing them; the buffer must then come from
     * that very forward, else no gradient is written and subq_device_status
     * reports SUBQ_ERR_STATE. */
    subq_tensor4 out;
} subq_bwd_args;

/* Forward scan. Replaces run_attention_forward / the torch chunked forward. */
int subq_fwd(const subq_fwd_args* args);

/* Backward scan (recomputes the forward; saves nothing between calls).
 * Replaces subquadratic_attention_backward / _single_direction_causal_backward. */
int subq_bwd(const subq_bwd_args* args);

/* Bytes of `workspace` the call needs (0 is possible). */
size_t subq_fwd_workspace_bytes(const subq_fwd_args* args);
size_t subq_bwd_workspace_bytes(const subq_bwd_args* args);
/* Bytes of the forward's optional segment_states buffer (0: the call would
 * not fill one, e.g. on the exact path). */
size_t subq_segment_states_bytes(const subq_fwd_args* args);

/* In-place phi(x) = ELU(x) + 1 over n contiguous elements (run_feature_map). */
int subq_feature_map(void* x, int64_t n, int32_t dtype, void* stream);

/* Per-head RMSNorm of the scan's output, y = x * rsqrt(mean_D(x^2) + eps) * w
 * over each row of D values (one token of one head): SubQLinearAttention's
 * nn.RMSNorm(head_dim, eps=1e-5) and the [B, H, L, D] -> [B, L, H*D] copy
 * after it (reference python/subq_audio/autograd.py:706-710, 763-769); y is
 * written through its own strides, so giving it the [B, L, H, D] layout
 * replaces the copy. Math in float32 whatever the dtype (fp32, fp16 or bf16).
 * x, y, dy and dx are [B, H, N, D] views with element strides; D is 8, 16,
 * 32, 64, 128 or 256 (SUBQ_ERR_UNSUPPORTED otherwise); every row starts on a
 * 16-byte boundary (data and strides). The backward reads x and dy and writes
 *   dx = r (dy w - xh mean_D(dy w xh)),  xh = x r,  r = rsqrt(mean_D(x^2) + eps)
 * and, when `dweight` is given, dweight = sum over rows of dy xh (written,
 * not accumulated; bitwise reproducible), which needs `workspace` of
 * subq_head_rmsnorm_bwd_workspace_bytes. dx may be x or dy (in place). */
typedef struct subq_rmsnorm_args {
    int64_t batch, heads, seq_len, head_dim;
    int32_t dtype;
    float eps;
    subq_tensor4 x, y;      /* forward: input and output (the backward reads x) */
    subq_tensor4 dy, dx;    /* backward: upstream gradient and input gradient */
    const float* weight;    /* [D] float32, or NULL for a weight of 1 */
    float* dweight;         /* backward: [D] float32, or NULL */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_rmsnorm_args;

int subq_head_rmsnorm_fwd(const subq_rmsnorm_args* args);
int subq_head_rmsnorm_bwd(const subq_rmsnorm_args* args);
size_t subq_head_rmsnorm_bwd_workspace_bytes(const subq_rmsnorm_args* args);

/* Gated delta rule (no counterpart in the reference): the scan whose update
 * corrects what the state already holds for a key instead of adding to it,
 *   S_t = gamma_t S_{t-1} + beta_t k_t (v_t - gamma_t S_{t-1}^T k_t)^T,
 *   o_t = scale S_t^T q_t,
 * per (batch, head) with S [d, e] float32, gamma_t = exp(log_gamma_t). A masked
 * token leaves S as it is, its o and gradients are 0, and nothing of its q, k,
 * v, dout, beta or log_gamma is used. q, k, v and o are [B, heads, N, *] views;
 * q, k and v may each have fewer heads (a divisor of `heads`), state head h
 * then reading head h / (heads / x_heads), and their gradients sum over the
 * group. fp32, fp16, bf16; products accumulate in float32, and operands in
 * between are carried to 24 bits of mantissa. For bounded states |k_t| <= 1
 * with beta_t in [0, 2] and gamma_t <= 1, as usual for the rule; the kernels do
 * not require it. A live token that is not finite makes its chunk of 64
 * tokens, and what follows, not finite.
 *
 * Paths: SUBQ_PATH_EXACT is the token-recurrent kernel (d, e <= 256),
 * SUBQ_PATH_CHUNKED the chunk kernels (d <= 128, e <= 256). AUTO takes the
 * recurrent kernel for d > 128 and for calls of at most 16 tokens that fill no
 * handover. The backward has the chunk form only (d <= 128).
 *
 * Memory, KB for each (batch, head) and 64 tokens (d = e = 64; d = e = 128), q, k,
 * v and o being 32 (64) in 16 bits and 64 (128) in float32:
 *   forward's workspace                32  (32), none with a handover
 *   handover                           80 (176)
 *   backward's workspace               48 (144) with a handover, 128 (320) without
 * Where a call with few sequences is cut into segments, 32 KB (128 KB above
 * d = 64) for each (batch, head) and segment; the backward also holds float32
 * gradients per state head of shared q, k and v. The recurrent kernel needs none. */
typedef struct subq_gate {
    const float* data; /* [B, heads, N] float32 with element strides (0 allowed) */
    int64_t stride_b, stride_h, stride_n;
} subq_gate;

typedef struct subq_delta_desc {
    int64_t batch, heads, seq_len, head_dim, value_dim;
    int64_t q_heads, k_heads, v_heads; /* 0: `heads` */
    int32_t dtype;
    int32_t path;           /* AUTO, EXACT or CHUNKED                          */
    float scale;
    subq_gate beta;         /* data NULL: 1                                    */
    subq_gate log_gamma;    /* data NULL: 0 (no decay)                         */
    const uint8_t* mask;    /* as in subq_scan_desc                            */
    int64_t mask_stride_b;
} subq_delta_desc;

typedef struct subq_delta_fwd_args {
    subq_delta_desc desc;
    subq_tensor4 q, k, v, o; /* o shares no memory with an input (views of one
                               buffer between each other are fine)             */
    const float* state_in;  /* [B, heads, d, e], NULL = zeros                  */
    float* state_out;       /* may equal state_in, NULL = not wanted           */
    void* handover;         /* NULL, or subq_delta_handover_bytes (256-byte aligned)
                               to keep for the backward of the same call       */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_delta_fwd_args;

typedef struct subq_delta_bwd_args {
    subq_delta_desc desc;
    subq_tensor4 q, k, v, dout;
    subq_tensor4 dq, dk, dv;     /* heads of q, k, v; no output shares memory with
                                    an input or with another output              */
    const float* state_in;       /* the forward's                                */
    const float* dstate_out;     /* gradient of the final state, NULL = zeros    */
    float* dstate_in;            /* gradient of state_in, NULL = not wanted; may
                                    equal dstate_out                              */
    float* dbeta;                /* [B, heads, N] contiguous float32             */
    float* dlog_gamma;           /* likewise, or NULL                            */
    const void* handover;        /* what the forward of the same call left, or
                                    NULL: formed again in the workspace          */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_delta_bwd_args;

int subq_delta_fwd(const subq_delta_fwd_args* args);
int subq_delta_bwd(const subq_delta_bwd_args* args);
size_t subq_delta_fwd_workspace_bytes(const subq_delta_fwd_args* args);
size_t subq_delta_bwd_workspace_bytes(const subq_delta_bwd_args* args);
size_t subq_delta_handover_bytes(const subq_delta_desc* desc);

/* Layer norm over the last dimension of [rows, dim] (rows at element strides,
 * elements contiguous): y = (x - mean) rsqrt(var + eps) weight + bias, as
 * torch's layer_norm, sums in float32. x_dtype and y_dtype are equal (fp32,
 * fp16, bf16), or x is fp32 and y fp16 or bf16; dx has x's type and dy has y's.
 * The backward recomputes the statistics from x; dweight = sum dy xh and
 * dbias = sum dy are written (not accumulated), bitwise reproducible. Outputs
 * share no memory with inputs or one another, but for y or dx in place. */
typedef struct subq_layer_norm_args {
    int64_t rows, dim;
    int32_t x_dtype, y_dtype;
    float eps;
    const void* x;  int64_t x_stride;
    void* y;        int64_t y_stride;   /* forward; may be x (of one type and stride) */
    const void* dy; int64_t dy_stride;  /* backward */
    void* dx;       int64_t dx_stride;  /* may be x or dy (of one type and stride) for dim <= 8192 */
    const float* weight;                /* [dim] or NULL (1) */
    const float* bias;                  /* [dim] or NULL (0) */
    float* dweight;                     /* [dim] or NULL */
    float* dbias;                       /* [dim] or NULL */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_layer_norm_args;

int subq_layer_norm_fwd(const subq_layer_norm_args* args);
int subq_layer_norm_bwd(const subq_layer_norm_args* args);
size_t subq_layer_norm_bwd_workspace_bytes(const subq_layer_norm_args* args);

/* Selective scan (no counterpart in the reference): per channel d of D and state
 * n of N, float32 states,
 *   dt_t = softplus(raw_t + dt_bias_d)            (softplus = 0: raw_t + dt_bias_d)
 *   h_t[n] = exp(dt_t A[d, n]) h_{t-1}[n] + dt_t u_t B_t[n]
 *   out_t = (sum_n C_t[n] h_t[n] + D_d u_t) silu(z_t)   (no z: without the last factor)
 * u, dt (raw), z and out are [B, L, D] views, B and C [B, L, G, N] views that the
 * D / G channels of a group share, all of one type (fp32, fp16, bf16) with
 * element strides and a contiguous innermost dimension. A masked token leaves h as
 * it is, its out and gradients are 0, and nothing of it is used. N <= 128.
 *
 * The forward can leave the states before every eighth token (handover) for the
 * backward of the same call, which forms them again without: 4 bytes x the states
 * rounded up to 16, 32, 64 or 128, for each channel and 8 tokens (8 bytes a token
 * and channel at N <= 16).
 *
 * The backward's workspace holds as much again without a handover, and the parts
 * of dB and dC: 8 n^2 / 1024 bytes a token and channel with n the states rounded up
 * as above (2 bytes at N <= 16, 8, 32, 128), but no more than 1 GiB or a float32
 * [B, L, D], whichever is more (or 32 tokens of each segment, where that is more):
 * beyond that the walk back goes in ranges of tokens, two launches each. */
typedef struct subq_tensor3 {
    void* data;
    int64_t stride_b, stride_l, stride_g; /* element strides; stride_g: B, C and their gradients only */
} subq_tensor3;

typedef struct subq_selective_desc {
    int64_t batch, seq_len, channels, states, groups;
    int32_t dtype;
    int32_t softplus;
    const float* A;         /* [channels, states]                              */
    const float* D;         /* [channels], or NULL (0)                         */
    const float* dt_bias;   /* [channels], or NULL (0)                         */
    const uint8_t* mask;    /* as in subq_scan_desc                            */
    int64_t mask_stride_b;
} subq_selective_desc;

typedef struct subq_selective_fwd_args {
    subq_selective_desc desc;
    subq_tensor3 u, dt, z, B, C;  /* z.data NULL: no gate                      */
    subq_tensor3 out;             /* shares no memory with an input             */
    const float* state_in;        /* [B, channels, states], NULL = zeros        */
    float* state_out;             /* may equal state_in, NULL = not wanted      */
    void* handover;               /* NULL, or subq_selective_scan_handover_bytes
                                     (256-byte aligned)                         */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_selective_fwd_args;

typedef struct subq_selective_bwd_args {
    subq_selective_desc desc;
    subq_tensor3 u, dt, z, B, C, dout;
    subq_tensor3 du, ddt, dz, dB, dC; /* like u, dt, z, B, C; no output shares memory
                                         with an input or another output        */
    const float* state_in;
    const float* dstate_out;      /* gradient of the final state, NULL = zeros  */
    float* dstate_in;             /* or NULL; may equal dstate_out              */
    float* dA;                    /* [channels, states]                         */
    float* dD;                    /* [channels], or NULL                        */
    float* ddt_bias;              /* [channels], or NULL                        */
    const void* handover;         /* what the forward of the same call left, or NULL */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_selective_bwd_args;

int subq_selective_scan_fwd(const subq_selective_fwd_args* args);
int subq_selective_scan_bwd(const subq_selective_bwd_args* args);
size_t subq_selective_scan_fwd_workspace_bytes(const subq_selective_fwd_args* args);
size_t subq_selective_scan_bwd_workspace_bytes(const subq_selective_bwd_args* args);
size_t subq_selective_scan_handover_bytes(const subq_selective_desc* desc);

/* Short causal convolution over [B, L, D], one filter of width 2, 3 or 4 a channel:
 *   pre_t = bias + sum_j weight[d, j] x_{t-width+1+j},   y_t = silu(pre_t) or pre_t.
 * Before the first token stand the width - 1 inputs of state_in (zeros without);
 * a masked token's input counts as 0, its y and dx are 0 and nothing of it is used;
 * state_out receives the width - 1 inputs up to the last live token (those of
 * state_in among them where there are fewer; state_in itself without a live
 * token). Sums in float32; weights and their gradients float32, written (not
 * accumulated) and bitwise reproducible. */
typedef struct subq_causal_conv_args {
    int64_t batch, seq_len, channels, width;
    int32_t dtype;
    int32_t silu;
    subq_tensor3 x, y;      /* forward: y shares no memory with an input        */
    subq_tensor3 dy, dx;    /* backward                                         */
    const float* weight;    /* [channels, width]                                */
    const float* bias;      /* [channels], or NULL (0)                          */
    const uint8_t* mask;
    int64_t mask_stride_b;
    const void* state_in;   /* [B, width - 1, channels] of x's type, or NULL    */
    void* state_out;        /* forward; may equal state_in, NULL = not wanted   */
    const void* dstate_out; /* backward: gradient of state_out, or NULL         */
    void* dstate_in;        /* backward: gradient of state_in, or NULL          */
    float* dweight;         /* backward: [channels, width]                      */
    float* dbias;           /* backward: [channels], or NULL                    */
    void* workspace;        /* backward                                         */
    size_t workspace_bytes;
    void* stream;
} subq_causal_conv_args;

int subq_causal_conv_fwd(const subq_causal_conv_args* args);
int subq_causal_conv_bwd(const subq_causal_conv_args* args);
size_t subq_causal_conv_bwd_workspace_bytes(const subq_causal_conv_args* args);

/* Root-mean-square norm over the last dimension of [rows, dim] with the residual's
 * addition: r = x + residual (rounded to r's type; without a residual r is x),
 *   y = r rsqrt(mean(r^2) + eps) weight.
 * Types (x, r, y): r_dtype is that of residual and r, x's or fp32; y_dtype is x's,
 * or for an fp32 x also fp16 or bf16, or SUBQ_E4M3: then every 128 columns of a row
 * have a float32 scale = max(amax |y|, 1e-30) / 448 in `scale` [rows, ceil(dim /
 * 128)] and y holds y / scale rounded to e4m3. norm = 0 leaves the norm out (y is
 * r weight: quantising alone). dim <= 16384. Outputs share no memory with an input or
 * one another, but for r in x's or residual's place (of one type and row stride).
 *
 * The backward is given r: dr = rsqrt(..) (g - xh mean(g xh)) + dr_next with g = dy
 * weight (dy of x's type), dx and dres are dr in x's and r's types (either may be
 * NULL), dweight = sum over rows of dy xh (written, bitwise reproducible). */
#define SUBQ_E4M3 4

typedef struct subq_rms_norm_args {
    int64_t rows, dim;
    int32_t x_dtype, r_dtype, y_dtype;
    float eps;
    int32_t norm;
    const void* x;        int64_t x_stride;
    const void* residual; int64_t residual_stride;  /* or NULL */
    void* r;              int64_t r_stride;          /* or NULL; the backward's input */
    void* y;              int64_t y_stride;
    float* scale;         int64_t scale_stride;
    const float* weight;                             /* [dim], or NULL (1) */
    const void* dy;       int64_t dy_stride;
    const void* dr_next;  int64_t dr_next_stride;    /* of r's type, or NULL */
    void* dx;             int64_t dx_stride;
    void* dres;           int64_t dres_stride;
    float* dweight;                                  /* [dim], or NULL */
    void* workspace;
    size_t workspace_bytes;
    void* stream;
} subq_rms_norm_args;

int subq_rms_norm_fwd(const subq_rms_norm_args* args);
int subq_rms_norm_bwd(const subq_rms_norm_args* args);
size_t subq_rms_norm_bwd_workspace_bytes(const subq_rms_norm_args* args);

/* Product of e4m3 matrices with float32 scales for every 1 x 128 of a and every
 * 128 x 128 of b:
 *   out[m, n] = bias[n] + sum_kb a_scale[m, kb] b_scale[n / 128, kb] sum_{k in kb} a[m, k] b[n, k]
 * (b as a linear layer's weight [N, K]). The rows of a and b start on 16-byte
 * boundaries (data and strides, in bytes); any M, N and K. Sums in float32; out is
 * fp32, fp16 or bf16 and shares no memory with an input. */
typedef struct subq_scaled_matmul_args {
    int64_t M, N, K;
    int32_t out_dtype;
    const void* a;        int64_t a_stride;
    const float* a_scale; int64_t a_scale_stride;  /* [M, ceil(K / 128)]             */
    const void* b;        int64_t b_stride;
    const float* b_scale; int64_t b_scale_stride;  /* [ceil(N / 128), ceil(K / 128)] */
    const float* bias;                             /* [N], or NULL                   */
    void* out;            int64_t out_stride;
    void* stream;
} subq_scaled_matmul_args;

int subq_scaled_matmul(const subq_scaled_matmul_args* args);

/* Backward scan with no allocation and no caller workspace (no counterpart in
 * the reference, whose backward allocates its scratch on every call). For
 * callers that may not supply or grow device memory per call, such as a
 * real-time audio callback or a host with a fixed device budget: the scratch
 * is a static 8 MiB device buffer of the library. A call fits when
 * subq_bwd_workspace_bytes(args) <= 8 MiB: the recomputing tensor-core path
 * takes 8 bytes per token-head (B x H x N; 1,048,576 token-heads), 12 with
 * per-token decay (plus 4 bytes per sequence) and on the float32 exact path
 * (699,050), 24 on the float64 exact path (349,525); the one-pass backward
 * (segment_states and out given) takes a fixed 16.6 KB per SM (about 2.5 MB on
 * a B200) whatever the length; grouped K/V adds dK and dV per query head.
 * Larger calls return SUBQ_ERR_WORKSPACE. `workspace` and `workspace_bytes` of
 * args are ignored. Nothing in the buffer needs to start at zero (what must,
 * the call clears itself). There is one buffer per device, so calls that
 * overlap in time on one device race: serialise them. The first call on a
 * device looks the buffer up with that device current; make it before
 * capturing any of the device's streams. Results equal subq_bwd's. */
int subq_bwd_noalloc(const subq_bwd_args* args);

/* Reads and clears (in one atomic step, ordered on `stream`) the device status
 * word of the current device, then synchronises `stream`: SUBQ_OK, or
 * SUBQ_ERR_TIMEOUT when a bounded device-side wait of a tensor-core kernel gave
 * up since the last query, or SUBQ_ERR_STATE when a backward was given the
 * segment_states of another call's forward (the outputs are then not valid).
 * Returns SUBQ_ERR_CUDA if the launch or the synchronisation fails. */
int subq_device_status(void* stream, int* status);

/* Diagnostic (no counterpart in the reference): launches one block whose
 * bounded device-side wait - the one every tensor-core kernel uses on its
 * pipeline barriers - waits on a barrier that nothing arrives at, with its
 * limit shortened to `polls` (1..2^20) polls. It gives up and records
 * SUBQ_ERR_TIMEOUT in the device status word, as a stalled kernel would, so
 * that a caller can test its handling of subq_device_status without a fault. */
int subq_selftest_wait_timeout(int polls, void* stream);

/* Kernel path the last successful subq_fwd / subq_bwd of this thread ran. */
int subq_last_path(void);

/* Number of device kernels the last successful call of this thread launched. */
int subq_last_launches(void);

/* Message of this thread's last failing call ("" if none). */
const char* subq_last_error(void);

int subq_abi_version(void);

/* Device description for get_device_info (reference python/bindings.cpp:37-65).
 * `arch` receives e.g. "SM 10.0" (NUL-terminated, at most arch_len bytes). */
int subq_device_info(int device, char* arch, size_t arch_len, size_t* memory_bytes,
                     int* bf16_supported);

#ifdef __cplusplus
} /* extern "C" */
#endif
