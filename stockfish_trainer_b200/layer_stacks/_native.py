"""ctypes binding of ``libnnue_ls.so`` (C ABI declared in include/nnue_ls.h).

Built in-tree by ``stockfish_trainer_b200.build``.  There is no fallback: if
the library cannot be loaded every entry point raises.
"""

from __future__ import annotations

import ctypes
import os
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import build as _build
from .._native import NativeError

_P, _I64, _I32, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float
_U64, _SZ = ctypes.c_uint64, ctypes.c_size_t

OK = 0
ERR_INVALID_ARGUMENT = -1
ERR_UNSUPPORTED = -2
ERR_WORKSPACE = -3
ERR_CUDA = -4
DEVERR_WAIT_TIMEOUT = 1
DEVERR_BAD_INDEX = 2
NORM_MAX_WIDTH = 65536
MAX_EXPERTS = 1024

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Linear(ctypes.Structure):
    _fields_ = [("rows", _I64), ("inputs", _I64), ("outputs", _I64), ("dtype", _I32), ("bias_dtype", _I32),
                ("activation", _I32), ("reserved", _I32), ("x", _P), ("weight", _P), ("bias", _P), ("residual", _P),
                ("ldx", _I64), ("ldw", _I64), ("ldr", _I64), ("out", _P), ("act_grad", _P), ("x_packed", _P),
                ("weight_packed", _P), ("grad_out", _P),
                ("ldg", _I64), ("grad_x", _P), ("grad_weight", _P), ("grad_bias", _P)]


class Norm(ctypes.Structure):
    _fields_ = [("rows", _I64), ("width", _I32), ("dtype", _I32), ("params_dtype", _I32), ("gate_dtype", _I32),
                ("kind", _I32), ("gate_mode", _I32), ("gate_sigmoid", _I32), ("scale_value", _F), ("eps", _F),
                ("reserved", _I32), ("x", _P), ("f", _P), ("gate", _P), ("post_weight", _P), ("post_bias", _P),
                ("scale", _P), ("pre_weight", _P), ("pre_bias", _P), ("y", _P), ("h", _P), ("stats", _P),
                ("grad_y", _P), ("grad_h", _P), ("grad_x", _P), ("grad_f", _P), ("grad_gate", _P),
                ("grad_post_weight", _P), ("grad_post_bias", _P), ("grad_scale", _P), ("grad_pre_weight", _P),
                ("grad_pre_bias", _P)]


class Route(ctypes.Structure):
    _fields_ = [("rows", _I64), ("experts", _I32), ("k", _I32), ("dtype", _I32), ("renormalize", _I32),
                ("logits", _P), ("ld", _I64), ("valid", _P), ("indices", _P), ("gates", _P), ("counts", _P),
                ("loss", _P), ("grad_gates", _P), ("grad_loss", _P), ("grad_logits", _P)]


_SIGNATURES = {
    "nnue_ls_version": (_I32, []),
    "nnue_ls_last_error": (ctypes.c_char_p, []),
    "nnue_ls_launch_count": (_U64, []),
    "nnue_ls_device_errors": (_I32, [ctypes.POINTER(ctypes.c_uint32), _I32]),
    "nnue_ls_set_wait_limit": (_U64, [_U64]),
    "nnue_ls_linear_saved_layout": (_SZ, [ctypes.POINTER(Linear), _I32, ctypes.POINTER(_I64)]),
    "nnue_ls_linear_forward_workspace_size": (_SZ, [ctypes.POINTER(Linear)]),
    "nnue_ls_linear_forward": (_I32, [ctypes.POINTER(Linear), _P, _SZ, _P]),
    "nnue_ls_linear_backward_workspace_size": (_SZ, [ctypes.POINTER(Linear)]),
    "nnue_ls_linear_backward": (_I32, [ctypes.POINTER(Linear), _P, _SZ, _P]),
    "nnue_ls_norm_forward": (_I32, [ctypes.POINTER(Norm), _P]),
    "nnue_ls_norm_backward_workspace_size": (_SZ, [ctypes.POINTER(Norm)]),
    "nnue_ls_norm_backward": (_I32, [ctypes.POINTER(Norm), _P, _SZ, _P]),
    "nnue_ls_route_forward_workspace_size": (_SZ, [ctypes.POINTER(Route)]),
    "nnue_ls_route_forward": (_I32, [ctypes.POINTER(Route), _P, _SZ, _P]),
    "nnue_ls_route_backward": (_I32, [ctypes.POINTER(Route), _P]),
}

_lib = None
_lock = threading.Lock()


def load(build_if_missing: bool | None = None) -> ctypes.CDLL:
    """Load (building first if allowed and needed) the native library."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if build_if_missing is None:
            build_if_missing = os.environ.get("NNUE_FT_NO_BUILD", "0") != "1"
        path = _build.build_layer_stacks() if build_if_missing else _build.LS_LIB_PATH
        if not os.path.exists(path):
            raise ImportError(
                f"{path} is missing: build it with `python -m stockfish_trainer_b200.build` "
                "(there is no non-native implementation of this path)")
        L = ctypes.CDLL(path)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def exported_symbols() -> list[str]:
    return list(_SIGNATURES)


def last_error() -> str:
    msg = load().nnue_ls_last_error()
    return msg.decode() if msg else ""


def launch_count() -> int:
    """Kernels launched by the library so far (process-wide)."""
    return int(load().nnue_ls_launch_count())


def device_errors(clear: bool = True) -> int:
    """Sticky device error flags of the current device (synchronises)."""
    flags = ctypes.c_uint32(0)
    check("nnue_ls_device_errors", load().nnue_ls_device_errors(ctypes.byref(flags), int(clear)))
    return int(flags.value)


def set_wait_limit(seconds: float) -> float:
    """How long a matrix kernel waits for its own copies and products before it gives up, raises DEVERR_WAIT_TIMEOUT and
    leaves NaN in what it has not formed (4 s at first; 0: at once).  Returns the limit so far."""
    if not 0 <= seconds < 2**34:
        raise ValueError(f"seconds must be in [0, 2^34), got {seconds}")
    return load().nnue_ls_set_wait_limit(round(seconds * 1e9)) / 1e9


def check(func: str, rc: int) -> None:
    if rc != OK:
        raise NativeError(func, rc, last_error())


_calls: dict = {}  # name -> (function, its workspace-size function or None)


def _lookup(func: str):
    lib = load()
    size = func + "_workspace_size"
    _calls[func] = found = (getattr(lib, func), getattr(lib, size) if size in _SIGNATURES else None)
    return found


def run(func: str, args: ctypes.Structure, like: torch.Tensor) -> None:
    """Enqueue ``func(args)`` on the current stream of ``like``'s device.  Where
    the call takes a workspace, it comes from PyTorch's caching allocator."""
    index = like.get_device()
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return run(func, args, like)
    fn, size = _calls.get(func) or _lookup(func)
    ref = ctypes.byref(args)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if size is None:
        rc = fn(ref, stream)
    else:
        nbytes = size(ref)
        # the caching allocator returns 512-byte aligned blocks; the ABI needs 256
        ws = like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        rc = fn(ref, None if ws is None else ws.data_ptr(), nbytes, stream)
    if rc != OK:
        check(func, rc)


def differentiates(grad: bool) -> bool:
    """Whether a call has to go through its autograd function: a gradient may be asked for (``grad``: of some argument),
    or forward-mode differentiation is on, which the functions refuse where an argument carries a tangent."""
    return grad and torch.is_grad_enabled() or forward_ad._current_level >= 0


def once(backward):
    """``once_differentiable`` that costs nothing unless a graph of the backward is asked for."""
    guarded = once_differentiable(backward)

    def wrapper(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return wrapper


def linear_saved(a: Linear, parts: int, like: torch.Tensor) -> tuple[torch.Tensor | None, tuple]:
    """The buffer a linear forward keeps for its backward (parts: 1 act'(z), 2 x,
    4 weight), entered in ``a``, and the parts' offsets in it; None if it needs none."""
    offsets = (_I64 * 3)()
    nbytes = (_lib or load()).nnue_ls_linear_saved_layout(ctypes.byref(a), parts, offsets)
    offsets = tuple(offsets)
    if not nbytes:
        return None, offsets
    saved = like.new_empty(nbytes, dtype=torch.uint8)
    place_saved(a, saved, offsets)
    return saved, offsets


def place_saved(a: Linear, saved: torch.Tensor, offsets) -> None:
    base = saved.data_ptr()
    a.act_grad, a.x_packed, a.weight_packed = [base + o if o >= 0 else None for o in offsets]


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def check_tensor(t: torch.Tensor, name: str, dtypes=DTYPES, index: int | None = None) -> int:
    """Refuses what is not a CUDA tensor of one of ``dtypes`` (on GPU ``index``); returns its GPU's index."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, got {t.dtype}")
    at = t.get_device()
    if at < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if index is not None and at != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    return at


# a type alone, and beside fp32: what parameters may have next to 16-bit tensors
ALONE = {dt: (dt,) for dt in DTYPES}
OR_F32 = {dt: (dt,) if dt == torch.float32 else (dt, torch.float32) for dt in DTYPES}


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of its last dimension's rows, with unit column stride
    and rows that do not overlap; copied only where the layout asks for it."""
    m = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if m.is_contiguous():
        return m
    if (m.stride(1) != 1 and m.shape[1] > 1) or (m.stride(0) < m.shape[1] and m.shape[0] > 1):
        return m.contiguous()
    return m


def row_stride(m: torch.Tensor) -> int:
    return max(m.stride(0), m.shape[1])
