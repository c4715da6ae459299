"""ctypes binding of the C ABI in include/kernels.hpp (libsubq_b200.so).

This is the binding a Python caller of the reference's kernel layer adds to
reach the B200 scan: plain pointers, sizes and a stream handle, no torch
types. The structures mirror the header field for field.
"""
from __future__ import annotations

import ctypes
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libsubq_b200.so")

SUBQ_OK = 0
SUBQ_ERR_INVALID_ARGUMENT = 1
SUBQ_ERR_ALIAS = 2
SUBQ_ERR_UNSUPPORTED = 3
SUBQ_ERR_CUDA = 4
SUBQ_ERR_TIMEOUT = 5
SUBQ_ERR_WORKSPACE = 6
SUBQ_ERR_STATE = 7

SUBQ_FP32, SUBQ_FP16, SUBQ_BF16, SUBQ_FP64, SUBQ_E4M3 = 0, 1, 2, 3, 4
SUBQ_DECAY_NONE, SUBQ_DECAY_SCALAR, SUBQ_DECAY_PER_HEAD, SUBQ_DECAY_PER_TOKEN = 0, 1, 2, 3
SUBQ_PATH_AUTO, SUBQ_PATH_EXACT, SUBQ_PATH_TENSORCORE, SUBQ_PATH_CHUNKED = 0, 1, 2, 3

# Every symbol include/kernels.hpp declares.
EXPORTED = (
    "subq_fwd", "subq_bwd", "subq_fwd_workspace_bytes", "subq_bwd_workspace_bytes",
    "subq_feature_map", "subq_last_path", "subq_last_launches", "subq_last_error",
    "subq_abi_version", "subq_device_info", "subq_device_status", "subq_bwd_noalloc",
    "subq_segment_states_bytes", "subq_selftest_wait_timeout",
    "subq_head_rmsnorm_fwd", "subq_head_rmsnorm_bwd", "subq_head_rmsnorm_bwd_workspace_bytes",
    "subq_delta_fwd", "subq_delta_bwd", "subq_delta_fwd_workspace_bytes", "subq_delta_bwd_workspace_bytes",
    "subq_delta_handover_bytes",
    "subq_layer_norm_fwd", "subq_layer_norm_bwd", "subq_layer_norm_bwd_workspace_bytes",
    "subq_selective_scan_fwd", "subq_selective_scan_bwd", "subq_selective_scan_fwd_workspace_bytes",
    "subq_selective_scan_bwd_workspace_bytes", "subq_selective_scan_handover_bytes",
    "subq_causal_conv_fwd", "subq_causal_conv_bwd", "subq_causal_conv_bwd_workspace_bytes",
    "subq_rms_norm_fwd", "subq_rms_norm_bwd", "subq_rms_norm_bwd_workspace_bytes",
    "subq_scaled_matmul",
)


class Tensor4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_b", ctypes.c_int64),
                ("stride_h", ctypes.c_int64), ("stride_n", ctypes.c_int64)]


class ScanDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("seq_len", ctypes.c_int64),
        ("head_dim", ctypes.c_int64), ("value_dim", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("normalize", ctypes.c_int32),
        ("scale", ctypes.c_float), ("clamp_min", ctypes.c_float),
        ("decay_mode", ctypes.c_int32), ("log_gamma_scalar", ctypes.c_float),
        ("log_gamma", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("mask_stride_b", ctypes.c_int64),
        ("flush_subnormal", ctypes.c_int32), ("path", ctypes.c_int32),
        ("kv_heads", ctypes.c_int64), ("reverse", ctypes.c_int32),
    ]


class FwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", ScanDesc), ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("o", Tensor4),
        ("state_in", ctypes.c_void_p), ("norm_in", ctypes.c_void_p),
        ("state_out", ctypes.c_void_p), ("norm_out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("stream", ctypes.c_void_p), ("segment_states", ctypes.c_void_p),
    ]


class BwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", ScanDesc), ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("dout", Tensor4),
        ("dq", Tensor4), ("dk", Tensor4), ("dv", Tensor4),
        ("state_in", ctypes.c_void_p), ("norm_in", ctypes.c_void_p),
        ("dlog_gamma", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("stream", ctypes.c_void_p), ("segment_states", ctypes.c_void_p),
        ("out", Tensor4),
    ]


class RmsArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("seq_len", ctypes.c_int64),
        ("head_dim", ctypes.c_int64), ("dtype", ctypes.c_int32), ("eps", ctypes.c_float),
        ("x", Tensor4), ("y", Tensor4), ("dy", Tensor4), ("dx", Tensor4),
        ("weight", ctypes.c_void_p), ("dweight", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("stream", ctypes.c_void_p),
    ]


class Gate(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_b", ctypes.c_int64),
                ("stride_h", ctypes.c_int64), ("stride_n", ctypes.c_int64)]


class DeltaDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("seq_len", ctypes.c_int64),
        ("head_dim", ctypes.c_int64), ("value_dim", ctypes.c_int64),
        ("q_heads", ctypes.c_int64), ("k_heads", ctypes.c_int64), ("v_heads", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("path", ctypes.c_int32), ("scale", ctypes.c_float),
        ("beta", Gate), ("log_gamma", Gate),
        ("mask", ctypes.c_void_p), ("mask_stride_b", ctypes.c_int64),
    ]


class DeltaFwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", DeltaDesc), ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("o", Tensor4),
        ("state_in", ctypes.c_void_p), ("state_out", ctypes.c_void_p), ("handover", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class DeltaBwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", DeltaDesc), ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("dout", Tensor4),
        ("dq", Tensor4), ("dk", Tensor4), ("dv", Tensor4),
        ("state_in", ctypes.c_void_p), ("dstate_out", ctypes.c_void_p), ("dstate_in", ctypes.c_void_p),
        ("dbeta", ctypes.c_void_p), ("dlog_gamma", ctypes.c_void_p), ("handover", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class LayerNormArgs(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("x_dtype", ctypes.c_int32), ("y_dtype", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64),
        ("dy", ctypes.c_void_p), ("dy_stride", ctypes.c_int64), ("dx", ctypes.c_void_p), ("dx_stride", ctypes.c_int64),
        ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class Tensor3(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_b", ctypes.c_int64),
                ("stride_l", ctypes.c_int64), ("stride_g", ctypes.c_int64)]


class SelectiveDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("seq_len", ctypes.c_int64), ("channels", ctypes.c_int64),
        ("states", ctypes.c_int64), ("groups", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("softplus", ctypes.c_int32),
        ("A", ctypes.c_void_p), ("D", ctypes.c_void_p), ("dt_bias", ctypes.c_void_p),
        ("mask", ctypes.c_void_p), ("mask_stride_b", ctypes.c_int64),
    ]


class SelectiveFwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", SelectiveDesc), ("u", Tensor3), ("dt", Tensor3), ("z", Tensor3), ("B", Tensor3), ("C", Tensor3),
        ("out", Tensor3), ("state_in", ctypes.c_void_p), ("state_out", ctypes.c_void_p), ("handover", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class SelectiveBwdArgs(ctypes.Structure):
    _fields_ = [
        ("desc", SelectiveDesc), ("u", Tensor3), ("dt", Tensor3), ("z", Tensor3), ("B", Tensor3), ("C", Tensor3),
        ("dout", Tensor3), ("du", Tensor3), ("ddt", Tensor3), ("dz", Tensor3), ("dB", Tensor3), ("dC", Tensor3),
        ("state_in", ctypes.c_void_p), ("dstate_out", ctypes.c_void_p), ("dstate_in", ctypes.c_void_p),
        ("dA", ctypes.c_void_p), ("dD", ctypes.c_void_p), ("ddt_bias", ctypes.c_void_p), ("handover", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class CausalConvArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("seq_len", ctypes.c_int64), ("channels", ctypes.c_int64), ("width", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("silu", ctypes.c_int32),
        ("x", Tensor3), ("y", Tensor3), ("dy", Tensor3), ("dx", Tensor3),
        ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("mask_stride_b", ctypes.c_int64),
        ("state_in", ctypes.c_void_p), ("state_out", ctypes.c_void_p), ("dstate_out", ctypes.c_void_p),
        ("dstate_in", ctypes.c_void_p), ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class RmsNormArgs(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("dim", ctypes.c_int64),
        ("x_dtype", ctypes.c_int32), ("r_dtype", ctypes.c_int32), ("y_dtype", ctypes.c_int32),
        ("eps", ctypes.c_float), ("norm", ctypes.c_int32),
        ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64),
        ("r", ctypes.c_void_p), ("r_stride", ctypes.c_int64), ("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64),
        ("scale", ctypes.c_void_p), ("scale_stride", ctypes.c_int64), ("weight", ctypes.c_void_p),
        ("dy", ctypes.c_void_p), ("dy_stride", ctypes.c_int64), ("dr_next", ctypes.c_void_p), ("dr_next_stride", ctypes.c_int64),
        ("dx", ctypes.c_void_p), ("dx_stride", ctypes.c_int64), ("dres", ctypes.c_void_p), ("dres_stride", ctypes.c_int64),
        ("dweight", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p),
    ]


class ScaledMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("M", ctypes.c_int64), ("N", ctypes.c_int64), ("K", ctypes.c_int64), ("out_dtype", ctypes.c_int32),
        ("a", ctypes.c_void_p), ("a_stride", ctypes.c_int64), ("a_scale", ctypes.c_void_p), ("a_scale_stride", ctypes.c_int64),
        ("b", ctypes.c_void_p), ("b_stride", ctypes.c_int64), ("b_scale", ctypes.c_void_p), ("b_scale_stride", ctypes.c_int64),
        ("bias", ctypes.c_void_p), ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("stream", ctypes.c_void_p),
    ]


class SubqError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load libsubq_b200.so, building it first if it is missing."""
    global _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                import importlib.util

                spec = importlib.util.spec_from_file_location(
                    "_subq_build", os.path.join(os.path.dirname(_HERE), "build.py"))
                mod = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(mod)
                mod.build_lib()
            lib = ctypes.CDLL(LIB_PATH)
            lib.subq_fwd.argtypes = [ctypes.POINTER(FwdArgs)]
            lib.subq_fwd.restype = ctypes.c_int
            lib.subq_bwd.argtypes = [ctypes.POINTER(BwdArgs)]
            lib.subq_bwd.restype = ctypes.c_int
            lib.subq_bwd_noalloc.argtypes = [ctypes.POINTER(BwdArgs)]
            lib.subq_bwd_noalloc.restype = ctypes.c_int
            lib.subq_fwd_workspace_bytes.argtypes = [ctypes.POINTER(FwdArgs)]
            lib.subq_fwd_workspace_bytes.restype = ctypes.c_size_t
            lib.subq_bwd_workspace_bytes.argtypes = [ctypes.POINTER(BwdArgs)]
            lib.subq_bwd_workspace_bytes.restype = ctypes.c_size_t
            lib.subq_segment_states_bytes.argtypes = [ctypes.POINTER(FwdArgs)]
            lib.subq_segment_states_bytes.restype = ctypes.c_size_t
            lib.subq_feature_map.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p]
            lib.subq_feature_map.restype = ctypes.c_int
            lib.subq_last_path.restype = ctypes.c_int
            lib.subq_last_launches.restype = ctypes.c_int
            lib.subq_last_error.restype = ctypes.c_char_p
            lib.subq_abi_version.restype = ctypes.c_int
            lib.subq_device_info.argtypes = [ctypes.c_int, ctypes.c_char_p, ctypes.c_size_t,
                                             ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_int)]
            lib.subq_device_info.restype = ctypes.c_int
            lib.subq_device_status.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]
            lib.subq_device_status.restype = ctypes.c_int
            lib.subq_selftest_wait_timeout.argtypes = [ctypes.c_int, ctypes.c_void_p]
            lib.subq_selftest_wait_timeout.restype = ctypes.c_int
            for name in ("subq_head_rmsnorm_fwd", "subq_head_rmsnorm_bwd"):
                getattr(lib, name).argtypes = [ctypes.POINTER(RmsArgs)]
                getattr(lib, name).restype = ctypes.c_int
            lib.subq_head_rmsnorm_bwd_workspace_bytes.argtypes = [ctypes.POINTER(RmsArgs)]
            lib.subq_head_rmsnorm_bwd_workspace_bytes.restype = ctypes.c_size_t
            for name, args in (("subq_delta_fwd", DeltaFwdArgs), ("subq_delta_bwd", DeltaBwdArgs),
                               ("subq_layer_norm_fwd", LayerNormArgs), ("subq_layer_norm_bwd", LayerNormArgs),
                               ("subq_selective_scan_fwd", SelectiveFwdArgs), ("subq_selective_scan_bwd", SelectiveBwdArgs),
                               ("subq_causal_conv_fwd", CausalConvArgs), ("subq_causal_conv_bwd", CausalConvArgs),
                               ("subq_rms_norm_fwd", RmsNormArgs), ("subq_rms_norm_bwd", RmsNormArgs),
                               ("subq_scaled_matmul", ScaledMatmulArgs)):
                getattr(lib, name).argtypes = [ctypes.POINTER(args)]
                getattr(lib, name).restype = ctypes.c_int
            for name, args in (("subq_delta_fwd_workspace_bytes", DeltaFwdArgs),
                               ("subq_delta_bwd_workspace_bytes", DeltaBwdArgs),
                               ("subq_delta_handover_bytes", DeltaDesc),
                               ("subq_layer_norm_bwd_workspace_bytes", LayerNormArgs),
                               ("subq_selective_scan_fwd_workspace_bytes", SelectiveFwdArgs),
                               ("subq_selective_scan_bwd_workspace_bytes", SelectiveBwdArgs),
                               ("subq_selective_scan_handover_bytes", SelectiveDesc),
                               ("subq_causal_conv_bwd_workspace_bytes", CausalConvArgs),
                               ("subq_rms_norm_bwd_workspace_bytes", RmsNormArgs)):
                getattr(lib, name).argtypes = [ctypes.POINTER(args)]
                getattr(lib, name).restype = ctypes.c_size_t
            _lib = lib
    return _lib


def check(rc: int) -> None:
    if rc != SUBQ_OK:
        msg = load().subq_last_error().decode(errors="replace")
        if rc in (SUBQ_ERR_INVALID_ARGUMENT, SUBQ_ERR_ALIAS):
            raise ValueError(msg)
        raise SubqError(rc, msg)


def fwd(args: FwdArgs) -> None:
    check(load().subq_fwd(ctypes.byref(args)))


def bwd(args: BwdArgs) -> None:
    check(load().subq_bwd(ctypes.byref(args)))


def bwd_noalloc(args: BwdArgs) -> None:
    """subq_bwd_noalloc: the backward with the library's static scratch."""
    check(load().subq_bwd_noalloc(ctypes.byref(args)))


def head_rmsnorm_fwd(args: RmsArgs) -> None:
    check(load().subq_head_rmsnorm_fwd(ctypes.byref(args)))


def head_rmsnorm_bwd(args: RmsArgs) -> None:
    check(load().subq_head_rmsnorm_bwd(ctypes.byref(args)))


def head_rmsnorm_bwd_workspace_bytes(args: RmsArgs) -> int:
    return int(load().subq_head_rmsnorm_bwd_workspace_bytes(ctypes.byref(args)))


def delta_fwd(args: DeltaFwdArgs) -> None:
    check(load().subq_delta_fwd(ctypes.byref(args)))


def delta_bwd(args: DeltaBwdArgs) -> None:
    check(load().subq_delta_bwd(ctypes.byref(args)))


def delta_fwd_workspace_bytes(args: DeltaFwdArgs) -> int:
    return int(load().subq_delta_fwd_workspace_bytes(ctypes.byref(args)))


def delta_bwd_workspace_bytes(args: DeltaBwdArgs) -> int:
    return int(load().subq_delta_bwd_workspace_bytes(ctypes.byref(args)))


def delta_handover_bytes(desc: DeltaDesc) -> int:
    return int(load().subq_delta_handover_bytes(ctypes.byref(desc)))


def layer_norm_fwd(args: LayerNormArgs) -> None:
    check(load().subq_layer_norm_fwd(ctypes.byref(args)))


def layer_norm_bwd(args: LayerNormArgs) -> None:
    check(load().subq_layer_norm_bwd(ctypes.byref(args)))


def layer_norm_bwd_workspace_bytes(args: LayerNormArgs) -> int:
    return int(load().subq_layer_norm_bwd_workspace_bytes(ctypes.byref(args)))


def selective_scan_fwd(args: SelectiveFwdArgs) -> None:
    check(load().subq_selective_scan_fwd(ctypes.byref(args)))


def selective_scan_bwd(args: SelectiveBwdArgs) -> None:
    check(load().subq_selective_scan_bwd(ctypes.byref(args)))


def selective_scan_fwd_workspace_bytes(args: SelectiveFwdArgs) -> int:
    return int(load().subq_selective_scan_fwd_workspace_bytes(ctypes.byref(args)))


def selective_scan_bwd_workspace_bytes(args: SelectiveBwdArgs) -> int:
    return int(load().subq_selective_scan_bwd_workspace_bytes(ctypes.byref(args)))


def selective_scan_handover_bytes(desc: SelectiveDesc) -> int:
    return int(load().subq_selective_scan_handover_bytes(ctypes.byref(desc)))


def causal_conv_fwd(args: CausalConvArgs) -> None:
    check(load().subq_causal_conv_fwd(ctypes.byref(args)))


def causal_conv_bwd(args: CausalConvArgs) -> None:
    check(load().subq_causal_conv_bwd(ctypes.byref(args)))


def causal_conv_bwd_workspace_bytes(args: CausalConvArgs) -> int:
    return int(load().subq_causal_conv_bwd_workspace_bytes(ctypes.byref(args)))


def rms_norm_fwd(args: RmsNormArgs) -> None:
    check(load().subq_rms_norm_fwd(ctypes.byref(args)))


def rms_norm_bwd(args: RmsNormArgs) -> None:
    check(load().subq_rms_norm_bwd(ctypes.byref(args)))


def rms_norm_bwd_workspace_bytes(args: RmsNormArgs) -> int:
    return int(load().subq_rms_norm_bwd_workspace_bytes(ctypes.byref(args)))


def scaled_matmul(args: ScaledMatmulArgs) -> None:
    check(load().subq_scaled_matmul(ctypes.byref(args)))


def fwd_workspace_bytes(args: FwdArgs) -> int:
    return int(load().subq_fwd_workspace_bytes(ctypes.byref(args)))


def bwd_workspace_bytes(args: BwdArgs) -> int:
    return int(load().subq_bwd_workspace_bytes(ctypes.byref(args)))


def segment_states_bytes(args: FwdArgs) -> int:
    return int(load().subq_segment_states_bytes(ctypes.byref(args)))


def device_status(stream: int = 0) -> int:
    """Synchronises `stream` and returns (and clears) the device status word."""
    st = ctypes.c_int(0)
    check(load().subq_device_status(ctypes.c_void_p(stream), ctypes.byref(st)))
    return int(st.value)


def selftest_wait_timeout(polls: int = 1000, stream: int = 0) -> None:
    """subq_selftest_wait_timeout: a bounded device-side wait that runs out."""
    check(load().subq_selftest_wait_timeout(int(polls), ctypes.c_void_p(stream)))


def last_path() -> int:
    return int(load().subq_last_path())


def last_launches() -> int:
    return int(load().subq_last_launches())
