"""libpixelsplat_ops.so (the C ABI of pixelsplat_ops.h, through ctypes) and _binding.so (the same operators as torch
functions: what the package calls).  No fallback: a missing library raises."""
from __future__ import annotations

import ctypes as C
import os

import torch  # noqa: F401  (its HIP runtime has to be in the process before the library is)

from .._lib import HipExtensionMissing

LIB_PATH = os.environ.get("PIXELSPLAT_OPS_LIB") or os.path.join(
    os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "libpixelsplat_ops.so")

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}


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
_binding = None


def load():
    """Loads the library (cached).  Raises HipExtensionMissing -- never falls back."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise HipExtensionMissing(f"{LIB_PATH} not found: build it with `python -m pixelsplat_amd.ops.build` "
                                  "(hipcc --offload-arch=gfx950). There is no non-HIP fallback for these operators.")
    lib = C.CDLL(LIB_PATH)
    for name, (result, arguments) in SIGNATURES.items():
        if not hasattr(lib, name):
            raise HipExtensionMissing(f"{LIB_PATH} does not export {name}")
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = result, arguments
    _lib = lib
    return lib


def binding():
    """The operators as torch functions (_binding.so, csrc/binding.cpp): cached, and as loud when it is missing."""
    global _binding
    if _binding is None:
        load()
        try:
            from . import _binding as module
        except ImportError as e:
            raise HipExtensionMissing(f"pixelsplat_amd/ops/_binding.so is missing or does not load ({e}): build it with "
                                      "`python -m pixelsplat_amd.ops.build`. There is no fallback.") from e
        _binding = module
    return _binding


def activation_code(op: str, name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"{op}: activation {name!r} is none of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]
