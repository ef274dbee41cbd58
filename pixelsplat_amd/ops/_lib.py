"""ctypes binding of libpixelsplat_ops.so (the C ABI of pixelsplat_ops.h) and what its operators share: the checks of
their arguments, the launch on a tensor's own device and the status codes.  No fallback: a missing library raises."""
from __future__ import annotations

import ctypes as C
import os

import torch
from torch import Tensor

from .._lib import HipExtensionMissing

LIB_PATH = os.environ.get("PIXELSPLAT_OPS_LIB") or os.path.join(
    os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "libpixelsplat_ops.so")

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}
STATUS = {-1: "bad argument (null or misaligned pointer, inconsistent descriptor)", -2: "workspace too small",
          -3: "HIP launch failed", -4: "unsupported configuration"}


class PsGroupNormDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("samples", "rows", "channels", "groups", "dtype", "activation",
                                         "param_f32")] + [("eps", C.c_float)] + [
        (n, C.c_int64) for n in ("x_sample_stride", "x_row_stride", "dy_sample_stride", "dy_row_stride")]


class PsGatedLinearDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("rows", "dim", "hidden", "dtype", "activation", "reserved")] + [
        (n, C.c_int64) for n in ("x_row_stride", "w_row_stride", "dh_row_stride")]


class PsRelativeAttentionDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("batch", "heads", "queries", "query_start", "grid_h", "grid_w", "dim", "dtype",
                                         "buckets", "table_f32")] + [("scale", C.c_float), ("reserved", C.c_int32)] + [
        (n, C.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides", "do_strides")] + [("mask_stride", C.c_int64)]


_vp, _size, _i32 = C.c_void_p, C.c_size_t, C.c_int32
_pn, _pg, _pa = (C.POINTER(t) for t in (PsGroupNormDesc, PsGatedLinearDesc, PsRelativeAttentionDesc))
# every symbol pixelsplat_ops.h declares: (result, arguments)
SIGNATURES = {
    "ps_group_norm_workspace_bytes": (_size, [_pn, _i32]),
    "ps_group_norm_forward": (C.c_int, [_pn] + [_vp] * 7 + [_size, _vp]),
    "ps_group_norm_backward": (C.c_int, [_pn] + [_vp] * 10 + [_size, _vp]),
    "ps_gated_linear_forward": (C.c_int, [_pg] + [_vp] * 9),
    "ps_gated_linear_backward_workspace_bytes": (_size, [_pg]),
    "ps_gated_linear_backward": (C.c_int, [_pg] + [_vp] * 14 + [_size, _vp]),
    "ps_relative_attention_workspace_bytes": (_size, [_pa, _i32]),
    "ps_relative_attention_forward": (C.c_int, [_pa] + [_vp] * 11 + [_size, _vp]),
    "ps_relative_attention_backward": (C.c_int, [_pa] + [_vp] * 14 + [_size, _vp]),
    "ps_ops_build_info": (C.c_char_p, []),
}

_lib = None


def load():
    """Loads the library (cached).  Raises HipExtensionMissing -- never falls back."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise HipExtensionMissing(f"{LIB_PATH} not found: build it with `python -m pixelsplat_amd.ops.build` "
                                  "(hipcc --offload-arch=gfx950). There is no non-HIP fallback for these operators.")
    lib = C.CDLL(LIB_PATH)          # torch is imported above: both resolve to the HIP runtime it ships
    for name, (result, arguments) in SIGNATURES.items():
        if not hasattr(lib, name):
            raise HipExtensionMissing(f"{LIB_PATH} does not export {name}")
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = result, arguments
    _lib = lib
    return lib


def call(name: str, device: torch.device, *args) -> None:
    """lib.name(*args, stream) on `device` and its current stream; tensors become pointers, a status becomes an error."""
    fn = getattr(_lib or load(), name)
    args = [a.data_ptr() if isinstance(a, Tensor) else a for a in args]
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError(f"{name} failed: {STATUS.get(rc, 'unknown status')} (PsStatus {rc})")


def check_tensors(op: str, first: Tensor, **others: Tensor | None) -> None:
    """`first` is a GPU tensor of a supported type; every other tensor is on its device."""
    if first.dtype not in DTYPES:
        raise TypeError(f"{op}: fp32, bf16 or fp16 tensors, got {first.dtype}")
    if not first.is_cuda:
        raise RuntimeError(f"{op} needs GPU tensors (no CPU fallback)")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{op}: {name} is on {t.device}, the input on {first.device}")


def activation_code(op: str, name: str, allowed=tuple(ACTIVATIONS)) -> int:
    if name not in allowed:
        raise ValueError(f"{op}: activation {name!r} is none of {', '.join(allowed)}")
    return ACTIVATIONS[name]


def wants_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
