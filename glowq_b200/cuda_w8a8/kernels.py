"""The 8-bit entry points of the kernel library (include/glowq_w8a8.h): descriptors, and calls on packed descriptors."""
from __future__ import annotations

import ctypes
import struct

import torch

from ..cuda_w4a16 import kernels as K

F16, F32, BF16 = 0, 1, 2
NORM_NONE, NORM_LAYER, NORM_RMS = 0, 1, 2
R_NONE, R_COMPUTE, R_LOAD, FRESH = K.R_NONE, K.R_COMPUTE, K.R_LOAD, 16
MAX_EXACT_K, MAX_RANK, MAX_TOKENS = 131071, 1024, 1 << 22
DTYPES = {torch.float16: F16, torch.float32: F32, torch.bfloat16: BF16}

_vp, _i64, _i32, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t


class Rows(ctypes.Structure):
    _fields_ = ([(n, _vp) for n in ("x", "residual", "weight", "bias", "hidden", "y", "codes", "scales", "mean", "rstd", "stream")]
                + [("eps", ctypes.c_double)]
                + [(n, _i64) for n in ("x_stride", "residual_stride", "hidden_stride", "y_stride", "code_stride")]
                + [(n, _i32) for n in ("M", "K", "dtype", "norm", "constant", "reserved")])


class LayerNormGrad(ctypes.Structure):
    _fields_ = ([(n, _vp) for n in ("h", "dy", "dh", "weight", "mean", "rstd", "dx", "dweight", "dbias", "workspace")]
                + [("workspace_bytes", _sz), ("stream", _vp)]
                + [(n, _i64) for n in ("h_stride", "dy_stride", "dh_stride", "dx_stride")]
                + [(n, _i32) for n in ("M", "K", "dtype", "reserved")])


class Linear(ctypes.Structure):
    _fields_ = ([(n, _vp) for n in ("x", "codes", "scales", "weight", "weight_scales", "bias", "r_x", "R", "r", "L", "out", "stream")]
                + [(n, _i64) for n in ("x_stride", "code_stride", "weight_stride", "r_x_stride", "R_stride", "r_stride", "L_stride",
                                       "out_stride")]
                + [(n, _i32) for n in ("M", "K", "OC", "rank", "x_dtype", "out_dtype", "r_mode")]
                + [("alpha", ctypes.c_float), ("reserved", _i64)])


# The same layouts for struct.pack, which takes a tenth of the time of filling a ctypes structure field by field.
pack_rows = struct.Struct("@11Pd5q6i")
pack_grad = struct.Struct("@10PNP4q4i")
pack_linear = struct.Struct("@12P8q7ifq")
assert (pack_rows.size, pack_grad.size, pack_linear.size) == tuple(ctypes.sizeof(c) for c in (Rows, LayerNormGrad, Linear))

EXPORTS = ("glowq_w8a8_quantize", "glowq_layer_norm_forward", "glowq_layer_norm_workspace_bytes", "glowq_layer_norm_backward",
           "glowq_w8a8_linear", "glowq_w8a8_right_factor", "glowq_w8a8_read_status")


class _Ext:
    """The library's 8-bit entry points; the calls take packed descriptors (bytes)."""

    def __init__(self):
        base = K.load_w4a16_extension()
        lib = base.lib
        missing = [n for n in EXPORTS if not hasattr(lib, n)]
        if missing:
            raise RuntimeError(f"{K.library_path()} lacks symbols {missing}; rebuild with `python -m glowq_b200.build`")
        call = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p)
        self.lib, self.check = lib, base.check
        self.quantize = call(("glowq_w8a8_quantize", lib))
        self.layer_norm_forward = call(("glowq_layer_norm_forward", lib))
        self.layer_norm_backward = call(("glowq_layer_norm_backward", lib))
        self.linear = call(("glowq_w8a8_linear", lib))
        self.right_factor = call(("glowq_w8a8_right_factor", lib))
        lib.glowq_layer_norm_workspace_bytes.restype = _sz
        lib.glowq_layer_norm_workspace_bytes.argtypes = [ctypes.c_int, ctypes.c_int]
        lib.glowq_w8a8_read_status.argtypes = [_vp]


_ext = None


def ext() -> _Ext:
    global _ext
    if _ext is None:
        _ext = _Ext()
    return _ext


_device_now = K.current_device
tracing = torch.jit.is_tracing
_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 0)


def refuse_trace():
    raise RuntimeError("the 8-bit path cannot be traced (torch.jit.trace, make_fx): a trace does not see its launches and would keep nothing "
                       "but the allocation of their outputs; capture a CUDA graph")


def _proxies() -> bool:
    return torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None


def call(fn, device: torch.device, desc: bytes, what: str) -> None:
    """``fn(desc)`` with ``device`` current.  (What a trace by ``torch.jit`` gives as sizes is refused where sizes are read.)"""
    if _modes() and _proxies():
        refuse_trace()
    if _device_now() == device.index:
        rc = fn(desc)
    else:
        with torch.cuda.device(device):
            rc = fn(desc)
    if rc:
        ext().check(rc, what)
