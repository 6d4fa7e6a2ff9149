"""deepfuse_amd -- MI355X-native fp8 Linear path of DeepFuse, Python side.

The product is the C ABI in ``include/df_capi.h`` implemented by
``deepfuse_amd/libdeepfuse_amd.so`` (hand-written HIP for gfx950).  This module
binds it with ctypes and offers thin helpers over torch device tensors (torch
is only the allocator and stream provider here).  Nothing in this package has
a CPU fallback: if the HIP library is missing, :func:`lib` raises.

Reference mapping (SensorVista/DeepFuse):
  - ``DType`` mirrors ``OnnxLoader::DType`` (dnn/utils/onnx_loader.cuh:16-22),
    extended with the 1-byte fp8 formats.
  - ``fc_forward`` / ``fc_backward`` mirror ``FullyConnectedLayer<T>::forward``
    / ``backward`` (dnn/layers/fully_connected_layer.cu:164-357) in fp8 compute.
"""
from __future__ import annotations

import array
import ctypes
import enum
import itertools
import math
import operator
import os
import re
import warnings

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdeepfuse_amd.so")
HEADER_PATH = os.path.join(os.path.dirname(_HERE), "include", "df_capi.h")


class DType(enum.IntEnum):
    FLOAT32 = 0
    HALF = 1
    INT8 = 2
    UINT8 = 3
    BFLOAT16 = 4
    FP8E4M3 = 5
    FP8E5M2 = 6
    INT32 = 7


class Fmt(enum.IntEnum):
    E4M3 = 0
    E5M2 = 1


FMAX = {Fmt.E4M3: 448.0, Fmt.E5M2: 57344.0}


class DFError(RuntimeError):
    """A C-ABI call returned a negative status."""

    def __init__(self, fn: str, status: int, msg: str):
        super().__init__(f"{fn} failed with status {status}: {msg}")
        self.status = status


_c_int, _c_i64, _c_sz, _c_f = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
_c_u32 = ctypes.c_uint32
_vp = ctypes.c_void_p

# name -> (restype, argtypes); every function declared in df_capi.h
_SIGS = {
    "df_last_error_string": (ctypes.c_char_p, []),
    "df_version": (_c_int, []),
    "df_device_arch_ok": (_c_int, []),
    "df_absmax_workspace_bytes": (_c_sz, []),
    "df_absmax_f32": (_c_int, [_vp, _c_i64, _vp, _vp, _c_sz, _vp]),
    "df_absmax_bf16": (_c_int, [_vp, _c_i64, _vp, _vp, _c_sz, _vp]),
    "df_absmax_scale_f32": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp, _vp, _c_sz, _vp]),
    "df_absmax_scale_bf16": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp, _vp, _c_sz, _vp]),
    "df_absmax_f16": (_c_int, [_vp, _c_i64, _vp, _vp, _c_sz, _vp]),
    "df_absmax_scale_f16": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp, _vp, _c_sz, _vp]),
    "df_compute_scale": (_c_int, [_vp, _c_int, _vp, _vp]),
    "df_hbm_probe_dst_bytes": (_c_sz, [_c_int, _c_int, _c_i64]),
    "df_hbm_probe": (_c_int, [_c_int, _c_int, _vp, _c_i64, _vp, _vp]),
    "df_quantize_f32_e4m3": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_quantize_f32_e5m2": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_quantize_bf16_e4m3": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_quantize_bf16_e5m2": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_dequantize_e4m3_f32": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_dequantize_e5m2_f32": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_dequantize_e4m3_bf16": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_dequantize_e5m2_bf16": (_c_int, [_vp, _c_i64, _vp, _vp, _vp]),
    "df_quantize_2d": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _c_int,
                                _vp, _c_int, _vp]),
    "df_quantize_2d_workspace_bytes": (_c_sz, [_c_int, _c_int]),
    "df_quantize_2d_colsum": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _c_int,
                                       _vp, _c_int, _vp, _vp, _c_sz, _vp]),
    "df_quantize_2d_jit_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int]),
    "df_quantize_2d_jit": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_int, _vp, _c_int, _vp,
                                    _vp, _c_sz, _vp]),
    "df_colsum": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _c_sz, _vp]),
    "df_quantize_2d_batch_workspace_bytes": (_c_sz, []),
    "df_quantize_2d_batch": (_c_int, [_c_int, _c_int, _vp, _vp, _vp, _c_int, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                      _c_sz, _vp]),
    "df_quantize_2d_batch_absmax": (_c_int, [_c_int, _c_int, _vp, _vp, _vp, _c_int, _vp, _vp, _vp, _vp, _vp, _vp,
                                             _vp]),
    "df_fp8_gemm_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int]),
    "df_fp8_gemm_fwd_absmax_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int]),
    "df_fp8_gemm_fwd_absmax": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _c_int, _vp,
                                        _c_int, _vp, _c_int, _c_int, _vp, _vp, _vp, _c_sz, _vp]),
    "df_fp8_gemm_nt": (_c_int, [_c_int, _vp, _c_int, _c_int, _vp, _c_int, _c_int, _c_int, _c_int,
                                _vp, _vp, _c_int, _vp, _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_fp8_gemm_nt_plan": (_c_int, [_c_int, _c_int, _c_int, _c_int, _c_int, _vp, _c_sz, _vp, _vp]),
    "df_fp8_gemm_fwd_timeline": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp, _vp,
                                          _c_int, _vp, _c_int, ctypes.POINTER(_c_int), _vp]),
    "df_fp8_gemm_fwd": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp,
                                 _c_int, _vp, _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_fp8_gemm_bwd_dx": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp,
                                    _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_fp8_gemm_bwd_dw": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp,
                                    _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_fp8_gemm_bwd_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int]),
    "df_fp8_gemm_bwd_plan": (_c_int, [_c_int, _c_int, _c_int, _c_sz, _vp, _vp]),
    "df_fp8_gemm_bwd": (_c_int, [_vp, _c_int, _vp, _c_int, _vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp,
                                 _vp, _vp, _c_int, _vp, _c_int, _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_fp8_gemm_bwd_absmax_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int]),
    "df_fp8_gemm_bwd_absmax": (_c_int, [_vp, _c_int, _vp, _c_int, _vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int,
                                        _vp, _vp, _vp, _c_int, _vp, _c_int, _c_int, _vp, _c_int, _c_int, _vp, _vp,
                                        _vp, _c_sz, _vp]),
    "df_fp8_experts_fwd": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_int, _vp,
                                    _c_int, _vp]),
    "df_fp8_experts_dx": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_int, _vp,
                                   _c_int, _vp]),
    "df_fp8_experts_dw": (_c_int, [_vp, _c_int, _vp, _c_int, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_int, _vp,
                                   _c_int, _vp]),
    "df_fill": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp]),
    "df_add": (_c_int, [_c_int, _vp, _vp, _vp, _c_i64, _vp]),
    "df_convert": (_c_int, [_c_int, _vp, _c_int, _vp, _c_i64, _vp]),
    "df_equal_mask": (_c_int, [_c_int, _vp, _vp, _vp, _c_i64, _vp]),
    "df_approx_equal_mask": (_c_int, [_c_int, _vp, _vp, _vp, _c_i64, _c_f, _vp]),
    "df_host_alloc": (_c_int, [_c_sz, ctypes.POINTER(_vp)]),
    "df_host_free": (_c_int, [_vp]),
    "df_streamer_create": (_c_int, [_c_int, _c_sz, ctypes.POINTER(_vp)]),
    "df_streamer_destroy": (_c_int, [_vp]),
    "df_streamer_load": (_c_int, [_vp, _vp, _c_sz, ctypes.POINTER(_c_int), ctypes.POINTER(_vp)]),
    "df_streamer_wait": (_c_int, [_vp, _c_int, _vp]),
    "df_streamer_release": (_c_int, [_vp, _c_int, _vp]),
    "df_streamer_slot": (_c_int, [_vp, _c_int, ctypes.POINTER(_vp)]),
    "df_streamer_copy_stream": (_c_int, [_vp, _c_int, ctypes.POINTER(_vp)]),
    "df_streamer_set_timing": (_c_int, [_vp, _c_int]),
    "df_streamer_copy_log": (_c_int, [_vp, _vp, _vp, _c_int, ctypes.POINTER(_c_int)]),
    "df_amax_history_init": (_c_int, [_vp, _c_int, _vp, _c_int, _vp, _vp]),
    "df_quantize_2d_delayed_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int, _c_int, _c_int]),
    "df_quantize_2d_delayed": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_int, _vp,
                                        _c_int, _vp, _c_int, _vp, _vp, _c_sz, _vp]),
    "df_quantize_2d_delayed_noalloc": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _c_int, _vp, _vp, _vp,
                                                _c_int, _vp, _c_int, _vp, _c_int, _vp, _vp]),
    "df_layernorm_workspace_bytes": (_c_sz, [_c_int, _c_int, _c_int, _c_int]),
    "df_layernorm": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _c_f, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_layernorm_quantize": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _c_f, _vp, _c_int, _c_int,
                                       _vp, _vp, _vp, _c_int, _vp, _c_int, _vp, _c_sz, _vp]),
    "df_layernorm_quantize_delayed": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _c_f, _vp, _c_int,
                                               _c_int, _vp, _vp, _vp, _c_int, _vp, _c_int, _vp, _c_int, _vp, _c_sz,
                                               _vp]),
    "df_layernorm_forward": (_c_int, [_c_int, _vp, _c_int, _c_int, _c_int, _vp, _c_int, _vp, _c_int, _vp, _vp, _c_f,
                                      _vp, _c_int, _vp, _vp, _vp]),
    "df_layernorm_backward_workspace_bytes": (_c_sz, [_c_int, _c_int]),
    "df_layernorm_backward": (_c_int, [_c_int, _vp, _c_int, _vp, _c_int, _c_int, _c_int, _vp, _vp, _vp, _c_f, _vp,
                                       _c_int, _vp, _c_int, _vp, _vp, _vp, _c_sz, _vp]),
    "df_grad_norm_workspace_bytes": (_c_sz, [_c_int, _vp]),
    "df_grad_norm_f32": (_c_int, [_vp, _vp, _c_int, _vp, _vp, _c_sz, _vp]),
    "df_clip_grad_norm_f32": (_c_int, [_vp, _vp, _c_int, _c_f, _vp, _vp, _c_sz, _vp]),
    "df_adam_update_f32": (_c_int, [_vp, _vp, _vp, _vp, _vp, _c_int, _c_f, _c_f, _c_f, _c_f, _c_f,
                                    _c_int, _vp, _c_f, _vp]),
    "df_adam_update_absmax_f32": (_c_int, [_vp, _vp, _vp, _vp, _vp, _c_int, _c_f, _c_f, _c_f, _c_f, _c_f,
                                           _c_int, _vp, _c_f, _vp, _vp]),
    "df_grad_norm": (_c_int, [_c_int, _vp, _vp, _c_int, _vp, _vp, _c_sz, _vp]),
    "df_adamw_scale_count": (_c_i64, [_c_i64]),
    "df_adamw_update": (_c_int, [_c_int, _vp, _vp, _c_int, _vp, _c_int, _vp, _vp, _vp, _vp, _c_int, _vp, _c_f, _c_f,
                                 _c_f, _c_f, _vp, _c_int, _vp, _vp, _vp, _c_f, _vp, _vp]),
    "df_adamw_update_dithered": (_c_int, [_c_int, _vp, _vp, _c_int, _vp, _c_int, _vp, _vp, _vp, _vp, _c_int, _vp, _c_f,
                                          _c_f, _c_f, _c_f, _vp, _c_int, _vp, _vp, _vp, _c_f, _vp, _c_u32, _vp]),
}

_lib = None


def header_functions() -> list[str]:
    """Names of the functions include/df_capi.h declares."""
    text = open(HEADER_PATH).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(df_[a-z0-9_]+)\s*\(", text)))


def lib() -> ctypes.CDLL:
    """Load libdeepfuse_amd.so (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(make -C deepfuse_amd); there is no CPU fallback")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def check(fn: str, status: int) -> None:
    if status != 0:
        msg = lib().df_last_error_string()
        raise DFError(fn, status, msg.decode() if msg else "")


def call(fn: str, *args) -> None:
    check(fn, getattr(lib(), fn)(*args))


# ----------------------------------------------------------------------------
# torch helpers (device memory + current stream); the compute is the C ABI
# ----------------------------------------------------------------------------
def _torch():
    import torch
    return torch


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    # the handle itself: building a torch Stream around it takes 2.8 us of a
    # call's 15
    C = _torch()._C
    return C._cuda_getCurrentRawStream(C._cuda_getDevice())


def _in_dtype(t) -> DType:
    torch = _torch()
    if t.dtype == torch.float32:
        return DType.FLOAT32
    if t.dtype == torch.bfloat16:
        return DType.BFLOAT16
    if t.dtype == torch.float16:
        return DType.HALF
    raise TypeError(f"unsupported input dtype {t.dtype}")


_ABSMAX_SCALE = {DType.FLOAT32: "df_absmax_scale_f32", DType.BFLOAT16: "df_absmax_scale_bf16",
                 DType.HALF: "df_absmax_scale_f16"}


_WS = {}


def _ws_key(device, tag: str):
    """Cached workspaces are kept per device and per stream (the current
    torch stream, the one the calls go to).  Calls on different streams
    never share one.  A workspace replaced by a larger one was allocated
    while its stream was current, and only that stream used it, so torch's
    allocator reuses its memory in that stream's order."""
    return (str(device), tag, _stream())


def _workspace(device):
    torch = _torch()
    key = _ws_key(device, "absmax")
    if key not in _WS:
        _WS[key] = torch.empty(lib().df_absmax_workspace_bytes(), dtype=torch.uint8, device=device)
    return _WS[key]


def absmax_scale(x, fmt: Fmt):
    """(absmax, scale) as 1-element fp32 device tensors, contract D1/D2."""
    torch = _torch()
    am = torch.empty(1, dtype=torch.float32, device=x.device)
    sc = torch.empty(1, dtype=torch.float32, device=x.device)
    ws = _workspace(x.device)
    call(_ABSMAX_SCALE[_in_dtype(x)], _ptr(x), x.numel(), int(fmt), _ptr(am), _ptr(sc), _ptr(ws), ws.numel(),
         _stream())
    return am, sc


def quantize(x, scale, fmt: Fmt):
    """Flat quantize of a contiguous fp32/bf16 tensor -> uint8 codes (same shape)."""
    torch = _torch()
    src = {DType.FLOAT32: "f32", DType.BFLOAT16: "bf16"}.get(_in_dtype(x))
    if src is None:  # the flat kernels take fp32 and bf16; df_quantize_2d also binary16
        raise TypeError(f"quantize: {x.dtype} has no flat kernel (use quantize_2d)")
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    fn = f"df_quantize_{src}_{'e4m3' if fmt == Fmt.E4M3 else 'e5m2'}"
    call(fn, _ptr(x), x.numel(), _ptr(scale), _ptr(q), _stream())
    return q


def dequantize(q, scale, fmt: Fmt, out_dtype):
    torch = _torch()
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dequantize: output {out_dtype} not supported (fp32 or bf16)")
    out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    dst = "f32" if out_dtype == torch.float32 else "bf16"
    fn = f"df_dequantize_{'e4m3' if fmt == Fmt.E4M3 else 'e5m2'}_{dst}"
    call(fn, _ptr(q), q.numel(), _ptr(scale), _ptr(out), _stream())
    return out


def round16(v: int) -> int:
    return (v + 15) // 16 * 16


def _scratch(device, nbytes: int, tag: str):
    torch = _torch()
    key = _ws_key(device, tag)
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)
        _WS[key] = ws
    return ws


def quantize_2d(x, scale, fmt: Fmt, want_q=True, want_qt=False, colsum=False):
    """2-D quantize into GEMM operand layout: returns (q [R, ceil16(C)],
    qt [C, ceil16(R)]) with zero padding (either may be None), plus the fp32
    column sums when colsum=True."""
    torch = _torch()
    rows, cols = x.shape
    q = torch.empty((rows, round16(cols)), dtype=torch.uint8, device=x.device) if want_q else None
    qt = torch.empty((cols, round16(rows)), dtype=torch.uint8, device=x.device) if want_qt else None
    ldq = q.shape[1] if q is not None else 0
    ldqt = qt.shape[1] if qt is not None else 0
    if not colsum:
        call("df_quantize_2d", int(_in_dtype(x)), _ptr(x), rows, cols, x.stride(0), int(fmt), _ptr(scale),
             _ptr(q), ldq, _ptr(qt), ldqt, _stream())
        return q, qt
    cs = torch.empty(cols, dtype=torch.float32, device=x.device)
    ws = _scratch(x.device, int(lib().df_quantize_2d_workspace_bytes(rows, cols)), "colsum")
    call("df_quantize_2d_colsum", int(_in_dtype(x)), _ptr(x), rows, cols, x.stride(0), int(fmt),
         _ptr(scale), _ptr(q), ldq, _ptr(qt), ldqt, _ptr(cs), _ptr(ws), ws.numel(), _stream())
    return q, qt, cs


def quantize_2d_jit(x, fmt: Fmt, want_q=True, want_qt=False, colsum=False):
    """absmax, scale and the 2-D quantize at that scale in one call
    (df_quantize_2d_jit): returns (absmax, scale, q, qt), plus the fp32
    column sums when colsum=True; x is contiguous."""
    torch = _torch()
    if not x.is_contiguous():
        raise ValueError("quantize_2d_jit: x must be contiguous")
    rows, cols = x.shape
    am = torch.empty(1, dtype=torch.float32, device=x.device)
    sc = torch.empty(1, dtype=torch.float32, device=x.device)
    q = torch.empty((rows, round16(cols)), dtype=torch.uint8, device=x.device) if want_q else None
    qt = torch.empty((cols, round16(rows)), dtype=torch.uint8, device=x.device) if want_qt else None
    cs = torch.empty(cols, dtype=torch.float32, device=x.device) if colsum else None
    ws = _scratch(x.device, int(lib().df_quantize_2d_jit_workspace_bytes(rows, cols, int(colsum))), "jit")
    call("df_quantize_2d_jit", int(_in_dtype(x)), _ptr(x), rows, cols, int(fmt), _ptr(am), _ptr(sc), _ptr(q),
         q.shape[1] if q is not None else 0, _ptr(qt), qt.shape[1] if qt is not None else 0, _ptr(cs), _ptr(ws),
         ws.numel(), _stream())
    return (am, sc, q, qt, cs) if colsum else (am, sc, q, qt)


def gemm_workspace(M: int, N: int, K: int, device):
    """Device workspace sized so split-K is never limited (cached per device
    and current stream, grown as needed)."""
    torch = _torch()
    nbytes = int(lib().df_fp8_gemm_workspace_bytes(M, N, K))
    key = _ws_key(device, "gemm")
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)
        _WS[key] = ws
    return ws


def gemm_nt(a_q, fmt_a: Fmt, b_q, fmt_b: Fmt, K: int, sa, sb, bias=None, out_dtype=None,
            split_k=True):
    """C[M,N] = (A[M,:K] . B[N,:K]^T) * sa * sb + bias on fp8 MFMA."""
    torch = _torch()
    out_dtype = out_dtype or torch.float32
    M, N = a_q.shape[0], b_q.shape[0]
    c = torch.empty((M, N), dtype=out_dtype, device=a_q.device)
    bias_dt = int(DType.FLOAT32) if bias is None else int(_in_dtype(bias))
    c_dt = int(_in_dtype(c))
    ws = gemm_workspace(M, N, K, a_q.device) if split_k else None
    call("df_fp8_gemm_nt", int(fmt_a), _ptr(a_q), a_q.stride(0), int(fmt_b), _ptr(b_q), b_q.stride(0),
         M, N, K, _ptr(sa), _ptr(sb), bias_dt, _ptr(bias), c_dt, _ptr(c), c.stride(0), _ptr(ws),
         ws.numel() if ws is not None else 0, _stream())
    return c


def gemm_fwd_absmax(x_q, w_q, K: int, sx, sw, bias=None, out_dtype=None, next_fmt: Fmt = Fmt.E4M3):
    """Y = X . W^T * sx * sw + bias (df_fp8_gemm_fwd_absmax): returns (Y,
    absmax of Y as stored, the rule-D1/D2 scale of Y for next_fmt); Y is
    bf16 (default), float16 or fp32."""
    torch = _torch()
    out_dtype = out_dtype or torch.bfloat16
    M, N = x_q.shape[0], w_q.shape[0]
    y = torch.empty((M, N), dtype=out_dtype, device=x_q.device)
    am = torch.empty(1, dtype=torch.float32, device=x_q.device)
    sc = torch.empty(1, dtype=torch.float32, device=x_q.device)
    nbytes = int(lib().df_fp8_gemm_fwd_absmax_workspace_bytes(M, N, K))
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x_q.device)
    bias_dt = int(DType.FLOAT32) if bias is None else int(_in_dtype(bias))
    call("df_fp8_gemm_fwd_absmax", _ptr(x_q), x_q.stride(0), _ptr(w_q), w_q.stride(0), M, N, K, _ptr(sx), _ptr(sw),
         bias_dt, _ptr(bias), int(_in_dtype(y)), _ptr(y), y.stride(0), int(next_fmt), _ptr(am), _ptr(sc), _ptr(ws),
         ws.numel(), _stream())
    return y, am, sc


class GemmKernel(enum.IntEnum):
    """DF_GEMM_KERNEL_* of include/df_capi.h."""
    PERSISTENT = 0
    TILED_DMA_256 = 1
    TILED_DMA_128 = 2
    TILED_REG_256 = 3
    TILED_REG_128 = 4
    PERSISTENT_NARROW = 5
    SMALL_16 = 6
    SMALL_32 = 7


def gemm_plan(M: int, N: int, K: int, lda: int, ldb: int, bias=None, ws_bytes: int = 0):
    """(GemmKernel, K slices) that df_fp8_gemm_nt takes for these arguments
    (SMALL_*: the waves of a block, which share the K steps);
    ``bias`` is the bias tensor the call would pass (its alignment counts)."""
    k, s = _c_int(), _c_int()
    call("df_fp8_gemm_nt_plan", M, N, K, lda, ldb, _ptr(bias), ws_bytes, ctypes.byref(k), ctypes.byref(s))
    return GemmKernel(k.value), s.value


def gemm_bwd(dy_q, wt_q, dyt_q, xt_q, M: int, N: int, K: int, sdy, sw, sx, dx_dtype=None, dw_dtype=None,
             workspace=True):
    """dX [M, K] and dW [N, K] of one Linear in one call (df_fp8_gemm_bwd):
    dy_q [M, >=N] and dyt_q [N, >=M] e5m2, wt_q [K, >=N] and xt_q [K, >=M]
    e4m3, as df_quantize_2d writes them."""
    torch = _torch()
    dx_dtype = dx_dtype or torch.float32
    dw_dtype = dw_dtype or torch.float32
    dev = dy_q.device
    dX = torch.empty((M, K), dtype=dx_dtype, device=dev)
    dW = torch.empty((N, K), dtype=dw_dtype, device=dev)
    dt = lambda t: int(_in_dtype(torch.empty(0, dtype=t)))
    ws = None
    if workspace:
        ws = _scratch(dev, max(int(lib().df_fp8_gemm_bwd_workspace_bytes(M, N, K)), 16), "gemm_bwd")
    call("df_fp8_gemm_bwd", _ptr(dy_q), dy_q.stride(0), _ptr(wt_q), wt_q.stride(0), _ptr(dyt_q), dyt_q.stride(0),
         _ptr(xt_q), xt_q.stride(0), M, N, K, _ptr(sdy), _ptr(sw), _ptr(sx), dt(dx_dtype), _ptr(dX), K,
         dt(dw_dtype), _ptr(dW), K, _ptr(ws), ws.numel() if ws is not None else 0, _stream())
    return dX, dW


def quantize_2d_batch(tensors, fmt: Fmt, want_q=True, want_qt=True, absmax=None):
    """df_quantize_2d_batch over contiguous 2-D device tensors (fp32 or
    bf16, one dtype): returns (absmax [count], scale [count], [q], [qt])
    with q [R, ceil16(C)] and qt [C, ceil16(R)] (None where not wanted).
    With ``absmax`` given (device fp32 [count]) the absmax pass is skipped
    (df_quantize_2d_batch_absmax) and that tensor is returned."""
    torch = _torch()
    count = len(tensors)
    dev = tensors[0].device
    am = torch.empty(count, dtype=torch.float32, device=dev) if absmax is None else absmax
    sc = torch.empty(count, dtype=torch.float32, device=dev)
    qs = [torch.empty((t.shape[0], round16(t.shape[1])), dtype=torch.uint8, device=dev) if want_q else None
          for t in tensors]
    qts = [torch.empty((t.shape[1], round16(t.shape[0])), dtype=torch.uint8, device=dev) if want_qt else None
           for t in tensors]
    arr = lambda vals: (_c_int * count)(*vals)
    ptrs = lambda ts: (_vp * count)(*[_ptr(t) for t in ts])
    head = (int(_in_dtype(tensors[0])), count, ptrs(tensors), arr([t.shape[0] for t in tensors]),
            arr([t.shape[1] for t in tensors]), int(fmt), _ptr(am), _ptr(sc))
    tail = (ptrs(qs) if want_q else None, arr([q.stride(0) for q in qs]) if want_q else None,
            ptrs(qts) if want_qt else None, arr([q.stride(0) for q in qts]) if want_qt else None)
    if absmax is None:
        ws = _scratch(dev, int(lib().df_quantize_2d_batch_workspace_bytes()), "qbatch")
        call("df_quantize_2d_batch", *head, *tail, _ptr(ws), ws.numel(), _stream())
    else:
        call("df_quantize_2d_batch_absmax", *head, *tail, _stream())
    return am, sc, qs, qts


def gemm_bwd_absmax(dy_q, wt_q, dyt_q, xt_q, M: int, N: int, K: int, sdy, sw, sx, dx_dtype=None, dw_dtype=None,
                    next_fmt: Fmt = Fmt.E5M2):
    """gemm_bwd whose dX also gives its absmax and the rule-D1/D2 scale for
    next_fmt (df_fp8_gemm_bwd_absmax): returns (dX, dW, absmax, scale)."""
    torch = _torch()
    dx_dtype = dx_dtype or torch.bfloat16
    dw_dtype = dw_dtype or torch.float32
    dev = dy_q.device
    dX = torch.empty((M, K), dtype=dx_dtype, device=dev)
    dW = torch.empty((N, K), dtype=dw_dtype, device=dev)
    am = torch.empty(1, dtype=torch.float32, device=dev)
    sc = torch.empty(1, dtype=torch.float32, device=dev)
    dt = lambda t: int(_in_dtype(torch.empty(0, dtype=t)))
    ws = _scratch(dev, max(int(lib().df_fp8_gemm_bwd_absmax_workspace_bytes(M, N, K)), 16), "gemm_bwd_absmax")
    call("df_fp8_gemm_bwd_absmax", _ptr(dy_q), dy_q.stride(0), _ptr(wt_q), wt_q.stride(0), _ptr(dyt_q),
         dyt_q.stride(0), _ptr(xt_q), xt_q.stride(0), M, N, K, _ptr(sdy), _ptr(sw), _ptr(sx), dt(dx_dtype), _ptr(dX),
         K, dt(dw_dtype), _ptr(dW), K, int(next_fmt), _ptr(am), _ptr(sc), _ptr(ws), ws.numel(), _stream())
    return dX, dW, am, sc


def gemm_bwd_plan(M: int, N: int, K: int, ws_bytes: int | None = None):
    """(grouped, dW slices) that df_fp8_gemm_bwd picks; ws_bytes defaults
    to df_fp8_gemm_bwd_workspace_bytes."""
    if ws_bytes is None:
        ws_bytes = int(lib().df_fp8_gemm_bwd_workspace_bytes(M, N, K))
    g, s = _c_int(), _c_int()
    call("df_fp8_gemm_bwd_plan", M, N, K, ws_bytes, ctypes.byref(g), ctypes.byref(s))
    return bool(g.value), s.value


def colsum(x):
    torch = _torch()
    rows, cols = x.shape
    out = torch.empty(cols, dtype=torch.float32, device=x.device)
    ws = _scratch(x.device, int(lib().df_quantize_2d_workspace_bytes(rows, cols)), "colsum")
    call("df_colsum", int(_in_dtype(x)), _ptr(x), rows, cols, x.stride(0), _ptr(out), _ptr(ws), ws.numel(),
         _stream())
    return out


class WeightStreamer:
    """Ring of device weight slots filled from pinned host memory on a copy
    stream (``df_streamer_*`` in include/df_capi.h).  ``load`` returns
    (slot, device pointer); ``wait`` / ``release`` order the slot against the
    current torch stream."""

    def __init__(self, slots: int, slot_bytes: int):
        h = _vp()
        call("df_streamer_create", slots, slot_bytes, ctypes.byref(h))
        self.handle = h
        self.slots = slots

    def load(self, host_ptr: int, nbytes: int):
        slot = _c_int()
        dev = _vp()
        call("df_streamer_load", self.handle, host_ptr, nbytes, ctypes.byref(slot), ctypes.byref(dev))
        return slot.value, dev.value

    def wait(self, slot: int, stream: int | None = None):
        call("df_streamer_wait", self.handle, slot, _stream() if stream is None else stream)

    def release(self, slot: int, stream: int | None = None):
        call("df_streamer_release", self.handle, slot, _stream() if stream is None else stream)

    def set_timing(self, on: bool = True):
        """Record HIP events around every later copy (see copy_log)."""
        call("df_streamer_set_timing", self.handle, 1 if on else 0)

    def copy_log(self) -> list[tuple[float, float]]:
        """(start, end) in ms of every timed copy since the last call, in load
        order (waits for them to finish); clears the log."""
        n = ctypes.c_int()
        call("df_streamer_copy_log", self.handle, None, None, 0, ctypes.byref(n))
        cap = n.value
        a, b = (ctypes.c_float * max(cap, 1))(), (ctypes.c_float * max(cap, 1))()
        call("df_streamer_copy_log", self.handle, a, b, cap, ctypes.byref(n))
        return [(a[i], b[i]) for i in range(min(cap, n.value))]

    def copy_streams(self) -> tuple[int, int]:
        """The two copy streams (load i runs on stream i % 2)."""
        out = []
        for which in (0, 1):
            st = _vp()
            call("df_streamer_copy_stream", self.handle, which, ctypes.byref(st))
            out.append(st.value or 0)
        return out[0], out[1]

    def close(self):
        if self.handle is not None:
            call("df_streamer_destroy", self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ----------------------------------------------------------------------------
# consumer side: global-norm clipping and Adam over lists of fp32 tensors
# (dnn/utils/clip_grad_norm.cu:31-67, dnn/optimizers/adam_optimizer.cu:11-109)
# ----------------------------------------------------------------------------
def _ptrs(tensors):
    return (_vp * max(len(tensors), 1))(*[t.data_ptr() for t in tensors])


def _sizes(tensors):
    return (_c_i64 * max(len(tensors), 1))(*[t.numel() for t in tensors])


def grad_norm(grads, clip: float | None = None):
    """Global L2 norm of fp32 device tensors as a 1-element device tensor;
    with ``clip`` the tensors are scaled in place by clip / norm when
    norm > clip (utils::clip_grad_norm).  bf16 and float16 tensors (one type
    for all) are measured too, without ``clip``."""
    torch = _torch()
    dev = grads[0].device
    if grads[0].dtype in (torch.bfloat16, torch.float16):
        return _grad_norm16(grads, clip)
    sizes = _sizes(grads)
    nbytes = lib().df_grad_norm_workspace_bytes(len(grads), sizes)
    ws = _scratch(dev, nbytes, "grad_norm")
    norm = torch.empty(1, dtype=torch.float32, device=dev)
    if clip is None:
        call("df_grad_norm_f32", _ptrs(grads), sizes, len(grads), _ptr(norm), _ptr(ws), ws.numel(), _stream())
    else:
        call("df_clip_grad_norm_f32", _ptrs(grads), sizes, len(grads), float(clip), _ptr(norm), _ptr(ws),
             ws.numel(), _stream())
    return norm


def adam_update(params, grads, ms, vs, timestep: int, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                weight_decay=0.0, clip_norm=None, max_norm=0.0, absmax=None):
    """One Adam step (AdamOptimizer<float>::step) over fp32 device tensors,
    in place on params, ms and vs; ``clip_norm`` (a device norm from
    :func:`grad_norm`) applies max_norm / norm to the gradients on the fly.
    ``absmax`` (an fp32 device tensor of len(params)) also receives max |p|
    of each updated tensor (df_adam_update_absmax_f32)."""
    n = len(params)
    assert len(grads) == n and len(ms) == n and len(vs) == n
    args = (_ptrs(params), _ptrs(grads), _ptrs(ms), _ptrs(vs), _sizes(params), n, float(lr), float(beta1),
            float(beta2), float(eps), float(weight_decay), int(timestep), _ptr(clip_norm), float(max_norm))
    if absmax is None:
        call("df_adam_update_f32", *args, _stream())
    else:
        assert absmax.numel() >= n and absmax.dtype == _torch().float32
        call("df_adam_update_absmax_f32", *args, _ptr(absmax), _stream())


# ----------------------------------------------------------------------------
# delayed scaling: scale from an amax history, absmax measured in the pass
# ----------------------------------------------------------------------------
class DelayedScale:
    """History and scale of one tensor role (fp32 device tensors)."""

    def __init__(self, fmt: Fmt, length: int, device, seed_amax=None):
        torch = _torch()
        self.fmt = Fmt(fmt)
        self.history = torch.empty(length, dtype=torch.float32, device=device)
        self.scale = torch.empty(1, dtype=torch.float32, device=device)
        call("df_amax_history_init", _ptr(seed_amax), int(self.fmt), _ptr(self.history), length,
             _ptr(self.scale), _stream())

    def quantize_2d(self, x, want_q=True, want_qt=False, colsum=False):
        """Like :func:`quantize_2d` with the current scale; returns
        (q, qt[, colsum]) and advances the history."""
        torch = _torch()
        rows, cols = x.shape
        q = torch.empty((rows, round16(cols)), dtype=torch.uint8, device=x.device) if want_q else None
        qt = torch.empty((cols, round16(rows)), dtype=torch.uint8, device=x.device) if want_qt else None
        ldq = q.shape[1] if q is not None else 0
        ldqt = qt.shape[1] if qt is not None else 0
        cs = torch.empty(cols, dtype=torch.float32, device=x.device) if colsum else None
        nbytes = lib().df_quantize_2d_delayed_workspace_bytes(rows, cols, ldq, ldqt, int(colsum))
        ws = _scratch(x.device, nbytes, "delayed")
        call("df_quantize_2d_delayed", int(_in_dtype(x)), _ptr(x), rows, cols, x.stride(0), int(self.fmt),
             _ptr(self.scale), _ptr(self.scale), _ptr(self.history), self.history.numel(), _ptr(q), ldq, _ptr(qt),
             ldqt, _ptr(cs), _ptr(ws), ws.numel(), _stream())
        return (q, qt, cs) if colsum else (q, qt)


# ----------------------------------------------------------------------------
# LayerNorm with the fused quantize (dnn/layers/layer_norm_layer.cu:26-63)
# ----------------------------------------------------------------------------
def layernorm(x, gamma=None, beta=None, eps=1e-5, fmt: Fmt | None = None, want_y=True, want_q=True,
              want_qt=False, delayed: "DelayedScale | None" = None):
    """LayerNorm over the last dim of a 2-D fp32/bf16 tensor.  fmt=None: y
    only.  Otherwise returns (y or None, q, qt, scale) with the codes of y at
    the just-in-time scale, or at ``delayed``'s history scale."""
    torch = _torch()
    rows, cols = x.shape
    dt = int(_in_dtype(x))
    y = torch.empty_like(x) if (want_y or fmt is None) else None
    ldy = cols if y is not None else 0
    if fmt is None:
        nbytes = lib().df_layernorm_workspace_bytes(rows, cols, 0, 0)
        ws = _scratch(x.device, nbytes, "layernorm")
        call("df_layernorm", dt, _ptr(x), rows, cols, x.stride(0), _ptr(gamma), _ptr(beta), float(eps), _ptr(y),
             ldy, _ptr(ws), ws.numel(), _stream())
        return y
    q = torch.empty((rows, round16(cols)), dtype=torch.uint8, device=x.device) if want_q else None
    qt = torch.empty((cols, round16(rows)), dtype=torch.uint8, device=x.device) if want_qt else None
    ldq = q.shape[1] if q is not None else 0
    ldqt = qt.shape[1] if qt is not None else 0
    nbytes = lib().df_layernorm_workspace_bytes(rows, cols, ldq, ldqt)
    ws = _scratch(x.device, nbytes, "layernorm")
    if delayed is None:
        scale = torch.empty(1, dtype=torch.float32, device=x.device)
        call("df_layernorm_quantize", dt, _ptr(x), rows, cols, x.stride(0), _ptr(gamma), _ptr(beta), float(eps),
             _ptr(y), ldy, int(fmt), _ptr(scale), None, _ptr(q), ldq, _ptr(qt), ldqt, _ptr(ws), ws.numel(),
             _stream())
    else:
        scale = delayed.scale.clone()
        call("df_layernorm_quantize_delayed", dt, _ptr(x), rows, cols, x.stride(0), _ptr(gamma), _ptr(beta),
             float(eps), _ptr(y), ldy, int(fmt), _ptr(scale), _ptr(delayed.scale), _ptr(delayed.history),
             delayed.history.numel(), _ptr(q), ldq, _ptr(qt), ldqt, _ptr(ws), ws.numel(), _stream())
    return y, q, qt, scale


# ----------------------------------------------------------------------------
# LayerNorm for training: the forward with its statistics, and the backward
# ----------------------------------------------------------------------------
class _on:
    """Context: the device of ``t`` is the current one, so that the call goes
    to that device's current stream."""

    __slots__ = ("at", "before")

    def __init__(self, t):
        self.at = t.get_device()

    def __enter__(self):
        self.before = _torch()._C._cuda_getDevice()
        if self.at != self.before:
            _torch().cuda.set_device(self.at)

    def __exit__(self, *exc):
        if self.at != self.before:
            _torch().cuda.set_device(self.before)


def _check_gpu(fn: str, **tensors):
    """Every given tensor is on one and the same GPU."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{fn}: {name} is on {t.device}, not on a GPU")
        at = t.get_device()
        if dev is not None and at != dev:
            raise ValueError(f"{fn}: {name} is on {t.device}, others on GPU {dev}")
        dev = at


_INT_MAX = 0x7FFFFFFF


def _fits(fn: str, *sizes: int):
    """Sizes and strides that the C interface can take: ctypes would cut a
    larger one to its low 32 bits.  (Asked where one of them, or-ed, is.)"""
    if max(sizes) > _INT_MAX:
        raise ValueError(f"{fn}: a size or stride of {max(sizes)}, past 32 bits")


def _check_like(fn: str, name: str, t, shape, dtype):
    if t.shape != shape or t.dtype is not dtype:
        raise ValueError(f"{fn}: {name} is {tuple(t.shape)} {t.dtype}, not {tuple(shape)} {dtype}")


def _rows(fn: str, name: str, t, shape, dtype) -> int:
    """The leading dimension of a [rows, cols] operand whose rows are
    contiguous and do not overlap."""
    _check_like(fn, name, t, shape, dtype)
    (rows, cols), (ld, step) = shape, t.stride()
    if cols > 1 and step != 1 or rows > 1 and ld < cols:
        raise ValueError(f"{fn}: {name} with strides {(ld, step)} has no contiguous rows of its own")
    if rows <= 1:
        return cols
    _fits(fn, ld)
    return ld


def _row_vector(fn: str, name: str, t, n: int, dtype):
    if t is not None:
        _check_like(fn, name, t, (n,), dtype)
        if n > 1 and t.stride(0) != 1:
            raise ValueError(f"{fn}: {name} is not contiguous")


def _plain(t, shape, dtype, at: int) -> bool:
    """Absent, or a contiguous tensor of this shape and type on GPU ``at``: the
    usual argument, seen in one test.  What is not gets its questions one by
    one, for the layouts allowed beyond this and the error's text."""
    return t is None or t.shape == shape and t.dtype is dtype and t.is_contiguous() and t.get_device() == at


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, residual=None):
    """LayerNorm over the last dim of a 2-D fp32/bf16/f16 tensor for training
    (df_layernorm_forward): returns (y, s, mean, rstd), where s = x + residual
    is what the norm saw (x itself without a residual) and mean and rstd are
    its rows' fp32 statistics: what :func:`layernorm_backward` takes."""
    fn, torch = "layernorm_forward", _torch()
    if x.dim() != 2:
        raise ValueError(f"{fn}: x has {x.dim()} dimensions, not 2")
    shape, dtype, at = x.shape, x.dtype, x.get_device()
    rows, cols = shape
    if (rows | cols) > _INT_MAX:
        _fits(fn, rows, cols)
    ldx = ldr = cols
    if not (at >= 0 and x.is_contiguous() and _plain(residual, shape, dtype, at) and _plain(gamma, (cols,), dtype, at)
            and _plain(beta, (cols,), dtype, at)):
        _check_gpu(fn, x=x, gamma=gamma, beta=beta, residual=residual)
        ldx = _rows(fn, "x", x, shape, dtype)
        ldr = cols if residual is None else _rows(fn, "residual", residual, shape, dtype)
        _row_vector(fn, "gamma", gamma, cols, dtype)
        _row_vector(fn, "beta", beta, cols, dtype)
    dt = _in_dtype(x)
    with _on(x):
        y = x.new_empty(shape)
        s = x if residual is None else x.new_empty(shape)
        mean = x.new_empty(rows, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        if cols == 0:  # the library writes nothing; a mean over no values is none
            mean.fill_(math.nan)
            rstd.fill_(math.nan)
        call("df_layernorm_forward", dt, x.data_ptr(), rows, cols, ldx, _ptr(residual), ldr,
             None if residual is None else s.data_ptr(), cols, _ptr(gamma), _ptr(beta), float(eps), y.data_ptr(), cols,
             mean.data_ptr(), rstd.data_ptr(), _stream())
    return y, s, mean, rstd


def layernorm_backward(dy, x, gamma=None, mean=None, rstd=None, eps=1e-5, dresidual=None, sums=True):
    """The gradients of :func:`layernorm_forward` (df_layernorm_backward), x
    being what the norm saw: returns (dx, dgamma, dbeta), the last two in fp32
    (None with ``sums=False``).  Without mean and rstd they are taken from x
    at eps again.  ``dresidual`` (the gradient that reaches the residual
    stream past the norm) is added to dx."""
    fn, torch = "layernorm_backward", _torch()
    if x.dim() != 2:
        raise ValueError(f"{fn}: x has {x.dim()} dimensions, not 2")
    shape, dtype, at = x.shape, x.dtype, x.get_device()
    rows, cols = shape
    if (rows | cols) > _INT_MAX:
        _fits(fn, rows, cols)
    ldx = lddy = lddr = cols
    if not (at >= 0 and x.is_contiguous() and _plain(dy, shape, dtype, at) and _plain(dresidual, shape, dtype, at)
            and _plain(gamma, (cols,), dtype, at) and _plain(mean, (rows,), torch.float32, at)
            and _plain(rstd, (rows,), torch.float32, at)):
        _check_gpu(fn, dy=dy, x=x, gamma=gamma, mean=mean, rstd=rstd, dresidual=dresidual)
        ldx, lddy = _rows(fn, "x", x, shape, dtype), _rows(fn, "dy", dy, shape, dtype)
        lddr = cols if dresidual is None else _rows(fn, "dresidual", dresidual, shape, dtype)
        _row_vector(fn, "gamma", gamma, cols, dtype)
        _row_vector(fn, "mean", mean, rows, torch.float32)
        _row_vector(fn, "rstd", rstd, rows, torch.float32)
    dt = _in_dtype(x)
    with _on(x):
        dx = x.new_empty(shape)
        dg = x.new_empty(cols, dtype=torch.float32) if sums else None
        db = torch.empty_like(dg) if sums else None
        # not a cached one: a captured graph keeps the workspace it was given
        nws = lib().df_layernorm_backward_workspace_bytes(rows, cols)
        ws = x.new_empty(nws, dtype=torch.uint8)
        call("df_layernorm_backward", dt, dy.data_ptr(), lddy, x.data_ptr(), ldx, rows, cols, _ptr(gamma), _ptr(mean),
             _ptr(rstd), float(eps), _ptr(dresidual), lddr, dx.data_ptr(), cols, _ptr(dg), _ptr(db), ws.data_ptr(), nws,
             _stream())
    return dx, dg, db


# ----------------------------------------------------------------------------
# AdamW over lists of tensors, states in 32 or in 8 bits
# ----------------------------------------------------------------------------
_dtype_of = operator.attrgetter("dtype")


def _lists(fn: str, at: int, lists):
    """Checks lists of contiguous tensors on GPU ``at``, given as (name,
    tensors, sizes, dtype), sizes one per parameter in each; returns all their
    addresses in order.  A map over all tensors per question: half the time of
    asking tensor by tensor."""
    T, n = _torch().Tensor, len(lists[0][2])
    every, want, dtypes = [], [], []
    for what, tensors, sizes, dtype in lists:
        if len(tensors) != n:
            raise ValueError(f"{fn}: {len(tensors)} {what} for {n} parameters")
        every += tensors
        want += sizes
        dtypes += [dtype] * n
    if not (list(map(T.numel, every)) == want and list(map(_dtype_of, every)) == dtypes
            and all(map(T.is_contiguous, every)) and set(map(T.get_device, every)) == {at}):
        for what, tensors, sizes, dtype in lists:
            for i, (t, k) in enumerate(zip(tensors, sizes)):
                if t.dtype != dtype or t.numel() != k or not t.is_contiguous() or t.get_device() != at:
                    raise ValueError(f"{fn}: {what}[{i}] ({tuple(t.shape)} {t.dtype} on {t.device}) is not a "
                                     f"contiguous {dtype} tensor of {k} values on GPU {at}")
    return array.array("Q", map(T.data_ptr, every))


def _grad_norm16(grads, clip):
    fn, torch = "grad_norm", _torch()
    if clip is not None:
        raise TypeError(f"{fn}: {grads[0].dtype} gradients are not clipped in place (give adamw_update the norm)")
    if not grads[0].is_cuda:
        raise ValueError(f"{fn}: the gradients are on {grads[0].device}, not on a GPU")
    _lists(fn, grads[0].get_device(), [("grads", grads, [t.numel() for t in grads], grads[0].dtype)])
    sizes = _sizes(grads)
    with _on(grads[0]):
        ws = torch.empty(int(lib().df_grad_norm_workspace_bytes(len(grads), sizes)), dtype=torch.uint8,
                         device=grads[0].device)
        norm = torch.empty(1, dtype=torch.float32, device=grads[0].device)
        call("df_grad_norm", int(_in_dtype(grads[0])), _ptrs(grads), sizes, len(grads), _ptr(norm), _ptr(ws), ws.numel(),
             _stream())
    return norm


def adamw_state(params, bits: int = 32):
    """(ms, vs, m_scales, v_scales) for :func:`adamw_update` before the first
    step: fp32 zeros and no scales (None), or with ``bits=8`` e4m3 zeros and
    an fp32 scale per 256 values (to be updated with ``dither``: see there)."""
    torch = _torch()
    if bits == 32:
        return [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params], None, None
    if bits != 8:
        raise ValueError(f"adamw_state: states in {bits} bits (8 or 32)")
    codes = lambda p: torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
    ones = lambda p: torch.ones(-(-p.numel() // 256), dtype=torch.float32, device=p.device)
    return ([codes(p) for p in params], [codes(p) for p in params], [ones(p) for p in params],
            [ones(p) for p in params])


_nearest_told = False


def _tell_nearest(fn: str):
    """Once a process: what 8-bit states without ``dither`` do."""
    global _nearest_told
    _nearest_told = True
    warnings.warn(f"{fn}: 8-bit states rounded to nearest do not follow v where it falls (steps stay too small); "
                  "give dither=<seed> to train", stacklevel=3)


def adamw_update(params, grads, ms, vs, timestep, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
                 m_scales=None, v_scales=None, copies=None, clip_norm=None, max_norm=0.0, absmax=None, dither=None):
    """One AdamW step (df_adamw_update) over contiguous fp32 parameters, in
    place on params, the states (fp32, or float8_e4m3fn with m_scales and
    v_scales: see :func:`adamw_state`) and ``copies`` (bf16 or float16, the
    updated parameters).  Gradients are fp32, bf16 or float16, one type for
    all.  ``weight_decay`` is one number or one per tensor; ``timestep`` an int
    or an int32 device tensor and ``lr`` a number or an fp32 device tensor,
    read when the kernel runs (a captured step follows them on replay).
    ``clip_norm`` (a device norm from :func:`grad_norm`, a tensor) applies
    max_norm / norm to the gradients where the norm is larger than max_norm,
    which then has to be above 0; ``absmax`` (fp32 of len(params)) receives
    max |p| of each updated tensor.

    ``dither`` (an int, the seed of the draws; it may stay the same, the step
    count is drawn on too) rounds 8-bit states up or down at random in proportion
    (df_adamw_update_dithered).  Without it they are rounded to nearest: exact
    for one step, but a root of v moves by at most (1 - beta2) / 2 a step, its
    codes lie 6 to 12% apart, and one that falls goes back to its code: after
    gradients have become smaller it stays too large (up to ten times after a
    tenfold fall), and the steps too small.  A training run gives ``dither``;
    the first call without it warns."""
    fn, torch = "adamw_update", _torch()
    n = len(params)
    if n == 0:
        return
    eight = m_scales is not None
    if eight != (v_scales is not None):
        raise ValueError(f"{fn}: m_scales and v_scales go together")
    if dither is not None and not eight:
        raise ValueError(f"{fn}: dither without 8-bit states")
    if eight and dither is None and not _nearest_told:
        _tell_nearest(fn)
    if not params[0].is_cuda:
        raise ValueError(f"{fn}: the parameters are on {params[0].device}, not on a GPU")
    gt = _in_dtype(grads[0]) if grads else DType.FLOAT32
    state = torch.float8_e4m3fn if eight else torch.float32
    sizes, at = [p.numel() for p in params], params[0].get_device()
    lists = [("params", params, sizes, torch.float32), ("grads", grads, sizes, grads[0].dtype if grads else None),
             ("ms", ms, sizes, state), ("vs", vs, sizes, state)]
    if eight:
        blocks = [-(-k // 256) for k in sizes]
        lists += [("m_scales", m_scales, blocks, torch.float32), ("v_scales", v_scales, blocks, torch.float32)]
    ct = DType.FLOAT32
    if copies is not None:
        ct = _in_dtype(copies[0]) if copies else ct
        if ct == DType.FLOAT32:
            raise TypeError(f"{fn}: copies are bf16 or float16")
        lists.append(("copies", copies, sizes, copies[0].dtype))
    addresses = _lists(fn, at, lists)
    written = addresses[:n] + addresses[2 * n:]  # all but the gradients
    if 0 in sizes:  # empty tensors share an address
        written = [a for a, k in zip(written, itertools.cycle(sizes)) if k]
    if len(set(written)) != len(written):
        raise ValueError(f"{fn}: a tensor that the step writes is listed twice")
    first = addresses.buffer_info()[0]
    p, g, m, v = (first + 8 * n * i for i in range(4))
    sm, sv = (first + 32 * n, first + 40 * n) if eight else (None, None)
    c = None if copies is None else first + 8 * n * (len(lists) - 1)
    if isinstance(weight_decay, (int, float)):
        wd = (_c_f * n)(*[weight_decay] * n)
    else:
        if len(weight_decay) != n:
            raise ValueError(f"{fn}: {len(weight_decay)} weight decays for {n} parameters")
        wd = (_c_f * n)(*weight_decay)
    scalars = {}
    for name, x, dt in (("timestep", timestep, torch.int32), ("lr", lr, torch.float32),
                        ("clip_norm", clip_norm, torch.float32)):
        if isinstance(x, torch.Tensor):
            if x.numel() != 1 or x.dtype != dt or x.device != params[0].device:
                raise ValueError(f"{fn}: {name} is not one {dt} on {params[0].device}")
            scalars[name] = x.data_ptr()
    if clip_norm is not None:
        if "clip_norm" not in scalars:
            raise TypeError(f"{fn}: clip_norm is a device norm (a tensor), not {type(clip_norm).__name__}")
        if not max_norm > 0:
            raise ValueError(f"{fn}: max_norm = {max_norm} with a clip_norm (a limit above 0)")
    if absmax is not None and (absmax.dtype != torch.float32 or absmax.numel() < n or not absmax.is_contiguous()
                               or absmax.device != params[0].device):
        raise ValueError(f"{fn}: absmax is not {n} contiguous fp32 values on {params[0].device}")
    with _on(params[0]):
        args = (n, (_c_i64 * n)(*sizes), p, gt, g, DType.FP8E4M3 if eight else DType.FLOAT32, m, v, sm,
                sv, ct, c, 0.0 if "lr" in scalars else float(lr), float(beta1), float(beta2), float(eps), wd,
                0 if "timestep" in scalars else int(timestep), scalars.get("lr"), scalars.get("timestep"),
                scalars.get("clip_norm"), float(max_norm), _ptr(absmax))
        if dither is None:
            call("df_adamw_update", *args, _stream())
        else:
            call("df_adamw_update_dithered", *args, int(dither) & 0xFFFFFFFF, _stream())


# ----------------------------------------------------------------------------
# products grouped by expert
# ----------------------------------------------------------------------------
def _codes_ld(fn: str, name: str, t) -> int:
    """The leading dimension of codes, a matrix or one per expert.  The stride
    of a dimension of one is arbitrary and says nothing."""
    rows, ld = t.shape[-2], t.stride(-2)
    if t.dim() == 3 and t.shape[0] > 1:
        if rows == 1:
            return t.stride(0)
        if t.stride(0) != rows * ld:
            raise ValueError(f"{fn}: the experts of {name} do not follow each other")
    return t.shape[-1] if rows == 1 and (ld < t.shape[-1] or ld % 16) else ld


def _experts_args(fn: str, offsets, scale, scales, experts: int, count: int, **codes):
    """Checks shared by the experts' products: devices, the offsets, the scales
    and the codes' layout; returns the codes' leading dimensions."""
    torch = _torch()
    at, (a, b) = offsets.get_device(), codes.values()
    if (at >= 0 and _plain(a, a.shape, torch.uint8, at) and _plain(b, b.shape, torch.uint8, at)
            and _plain(offsets, (experts + 1,), torch.int32, at) and scale.numel() == 1
            and _plain(scale, scale.shape, torch.float32, at) and scales.numel() == count
            and _plain(scales, scales.shape, torch.float32, at)):
        lda, ldb = a.shape[-1], b.shape[-1]
        if not (lda % 16 or ldb % 16):
            return lda, ldb
    _check_gpu(fn, offsets=offsets, scale=scale, scales=scales, **codes)
    _row_vector(fn, "offsets", offsets, experts + 1, torch.int32)
    for name, t, n in (("scale", scale, 1), ("scales", scales, count)):
        if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{fn}: the {name} {tuple(t.shape)} {t.dtype} is not {n} contiguous fp32 values")
    for name, t in codes.items():
        if t.dtype != torch.uint8 or t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{fn}: {name} is not uint8 codes with contiguous rows")
    return tuple(_codes_ld(fn, name, t) for name, t in codes.items())


def _experts_out(fn: str, out, shape, dtype, like):
    if out is None:
        return like.new_empty(shape, dtype=dtype or _torch().bfloat16), shape[-1]
    device = like.device
    if tuple(out.shape) != tuple(shape) or (dtype is not None and out.dtype != dtype) or out.device != device:
        raise ValueError(f"{fn}: out is {tuple(out.shape)} {out.dtype} on {out.device}, not {tuple(shape)} on {device}")
    if out.dim() == 2:
        return out, _rows(fn, "out", out, shape, out.dtype)
    if not out.is_contiguous():
        raise ValueError(f"{fn}: out is not contiguous")
    return out, shape[-1]


def _experts_rows(fn: str, c_fn: str, a_q, w_q, offsets, red: int, sa, sw, out_dtype, out):
    if a_q.dim() != 2 or w_q.dim() != 3:
        raise ValueError(f"{fn}: codes of {a_q.dim()} and {w_q.dim()} dimensions, not 2 and 3")
    experts, cols = w_q.shape[0], w_q.shape[1]
    lda, ldw = _experts_args(fn, offsets, sa, sw, experts, experts, rows=a_q, weights=w_q)
    if a_q.shape[1] < red or w_q.shape[2] < red:
        raise ValueError(f"{fn}: rows of {a_q.shape[1]} and {w_q.shape[2]} codes, fewer than {red}")
    rows = a_q.shape[0]
    if (rows | cols | red | experts | lda | ldw) > _INT_MAX:
        _fits(fn, rows, cols, red, experts, lda, ldw)
    out, ld = _experts_out(fn, out, (rows, cols), out_dtype, a_q)
    n, k = (cols, red) if c_fn == "df_fp8_experts_fwd" else (red, cols)
    with _on(a_q):
        call(c_fn, a_q.data_ptr(), lda, w_q.data_ptr(), ldw, rows, n, k, experts,
             offsets.data_ptr(), sa.data_ptr(), sw.data_ptr(), _in_dtype(out), out.data_ptr(), ld, _stream())
    return out


def experts_fwd(x_q, w_q, offsets, K: int, sx, sw, out_dtype=None, out=None):
    """Y [rows, N] of a Linear dealt to experts (df_fp8_experts_fwd): x_q
    [rows, >=K] and w_q [experts, N, >=K] e4m3 codes, zero from K to the next
    multiple of 16 as the quantize calls leave them, offsets int32
    [experts + 1] (expert e has rows offsets[e] to offsets[e+1], on the
    device), sx one scale, sw one per expert.  ``out`` keeps its rows that
    belong to no expert; a new output (bf16 unless out_dtype says otherwise)
    has them undefined."""
    return _experts_rows("experts_fwd", "df_fp8_experts_fwd", x_q, w_q, offsets, K, sx, sw, out_dtype, out)


def experts_dx(dy_q, wt_q, offsets, N: int, sdy, sw, out_dtype=None, out=None):
    """dX [rows, K] (df_fp8_experts_dx): dy_q [rows, >=N] e5m2 codes, wt_q
    [experts, K, >=N] the transposed e4m3 codes of each expert's weights, both
    zero from N to the next multiple of 16."""
    return _experts_rows("experts_dx", "df_fp8_experts_dx", dy_q, wt_q, offsets, N, sdy, sw, out_dtype, out)


def experts_dw(dyt_q, xt_q, offsets, rows: int, sdy, sx, out_dtype=None, out=None):
    """dW [experts, N, K] (df_fp8_experts_dw; fp32 unless out_dtype or ``out``
    says otherwise): dyt_q [N, >=rows] e5m2 and xt_q [K, >=rows] e4m3, the
    transposed codes of all rows."""
    fn, torch = "experts_dw", _torch()
    if dyt_q.dim() != 2 or xt_q.dim() != 2:
        raise ValueError(f"{fn}: codes of {dyt_q.dim()} and {xt_q.dim()} dimensions, not 2")
    if offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError(f"{fn}: offsets {tuple(offsets.shape)} are not experts + 1 values")
    experts = offsets.numel() - 1
    lddy, ldx = _experts_args(fn, offsets, sdy, sx, experts, 1, dyt_q=dyt_q, xt_q=xt_q)
    if dyt_q.shape[1] < rows or xt_q.shape[1] < rows:
        raise ValueError(f"{fn}: rows of {dyt_q.shape[1]} and {xt_q.shape[1]} codes, fewer than {rows}")
    N, K = dyt_q.shape[0], xt_q.shape[0]
    if (rows | N | K | experts | lddy | ldx) > _INT_MAX:
        _fits(fn, rows, N, K, experts, lddy, ldx)
    if out is None and out_dtype is None:
        out_dtype = torch.float32
    out, _ = _experts_out(fn, out, (experts, N, K), out_dtype, dyt_q)
    with _on(dyt_q):
        call("df_fp8_experts_dw", dyt_q.data_ptr(), lddy, xt_q.data_ptr(), ldx, rows, N, K, experts,
             offsets.data_ptr(), sdy.data_ptr(), sx.data_ptr(), _in_dtype(out), out.data_ptr(), K, _stream())
    return out


def quantize_experts(w, fmt: Fmt = Fmt.E4M3, want_q=True, want_qt=True):
    """Codes of the experts' weights w [experts, N, K] (contiguous fp32, bf16
    or float16) at a just-in-time scale per expert, laid out for the products
    above: returns (scales [experts], q [experts, N, ceil16(K)] or None, qt
    [experts, K, ceil16(N)] or None)."""
    fn, torch = "quantize_experts", _torch()
    if w.dim() != 3 or not w.is_contiguous():
        raise ValueError(f"{fn}: w {tuple(w.shape)} is not [experts, N, K] and contiguous")
    if not (want_q or want_qt):
        raise ValueError(f"{fn}: no codes wanted")
    _check_gpu(fn, w=w)
    E, N, K = w.shape
    _fits(fn, E, N, K)
    dt = int(_in_dtype(w))
    if w.numel() == 0:  # nothing to measure: the rule's scale of no values is 1
        none = lambda r, c: torch.zeros((E, r, round16(c)), dtype=torch.uint8, device=w.device)
        return (torch.ones(E, dtype=torch.float32, device=w.device), none(N, K) if want_q else None,
                none(K, N) if want_qt else None)
    with _on(w):
        src = w.view(E, N * K)
        if N * K * w.element_size() % 16 or w.data_ptr() % 16:  # the quantize calls take tensors at 16-byte boundaries
            src = w.new_empty((E, round16(N * K)))
            src[:, :N * K].copy_(w.view(E, N * K))
        new = lambda r, c: torch.empty((E, r, round16(c)), dtype=torch.uint8, device=w.device)
        q, qt = new(N, K) if want_q else None, new(K, N) if want_qt else None
        sc = torch.empty(E, dtype=torch.float32, device=w.device)
        ldq, ldqt = round16(K) if want_q else 0, round16(N) if want_qt else 0
        if w.dtype == torch.float16:  # the batched quantize takes fp32 and bf16
            ws = torch.empty(int(lib().df_quantize_2d_jit_workspace_bytes(N, K, 0)), dtype=torch.uint8, device=w.device)
            for e in range(E):
                call("df_quantize_2d_jit", dt, _ptr(src[e]), N, K, int(fmt), None, _ptr(sc[e:]),
                     _ptr(q[e]) if want_q else None, ldq, _ptr(qt[e]) if want_qt else None, ldqt, None, _ptr(ws),
                     ws.numel(), _stream())
            return sc, q, qt
        am = torch.empty(E, dtype=torch.float32, device=w.device)
        ws = torch.empty(int(lib().df_quantize_2d_batch_workspace_bytes()), dtype=torch.uint8, device=w.device)
        arr, ptrs = lambda v: (_c_int * E)(*[v] * E), lambda t: (_vp * E)(*[x.data_ptr() for x in t])
        call("df_quantize_2d_batch", dt, E, ptrs(src), arr(N), arr(K), int(fmt), _ptr(am), _ptr(sc),
             ptrs(q) if want_q else None, arr(ldq) if want_q else None, ptrs(qt) if want_qt else None,
             arr(ldqt) if want_qt else None, _ptr(ws), ws.numel(), _stream())
    return sc, q, qt
