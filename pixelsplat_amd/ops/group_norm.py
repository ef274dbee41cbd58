"""Group norm with an activation on channels-last maps (csrc/group_norm.hip)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch import Tensor, nn

from . import _lib


def _rows_view(x: Tensor) -> Tensor:
    """[n, rows, c] with unit channel stride: a view where the strides allow one, a copy otherwise."""
    n, c = x.shape[0], x.shape[-1]
    try:
        v = x.view(n, -1, c) if x.dim() != 3 else x
    except RuntimeError:
        v = x.reshape(n, -1, c)
    # the kernels read [n][rows][c] at positive strides
    if (c > 1 and v.stride(2) != 1) or (v.shape[1] > 1 and v.stride(1) < c):
        v = v.contiguous()
    return v


def _desc(x: Tensor, groups: int, eps: float, act: int, param: Optional[Tensor], dy: Optional[Tensor] = None):
    n, s, c = x.shape
    row = lambda t: t.stride(1) if s > 1 else c  # noqa: E731
    return _lib.PsGroupNormDesc(
        n, s, c, groups, _lib.DTYPES[x.dtype], act, int(param is not None and param.dtype == torch.float32), eps,
        x.stride(0) if n > 1 else 0, row(x), dy.stride(0) if dy is not None and n > 1 else 0,
        row(dy) if dy is not None else 0)


def _workspace(desc, backward: bool, device) -> tuple[Tensor, int]:
    size = _lib.load().ps_group_norm_workspace_bytes(C.byref(desc), int(backward))
    if size == 0:
        raise RuntimeError("group_norm: more than 8192 channels, 65535 samples or 2^31 elements in a sample")
    return torch.empty((size,), dtype=torch.uint8, device=device), size


def _forward(x: Tensor, groups: int, weight, bias, eps: float, act: int):
    """x [n, rows, c] -> (y contiguous, mean, rstd)"""
    n, s, c = x.shape
    y = torch.empty((n, s, c), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, n, groups), dtype=torch.float32, device=x.device)
    desc = _desc(x, groups, eps, act, weight if weight is not None else bias)
    ws, size = _workspace(desc, False, x.device)
    _lib.call("ps_group_norm_forward", x.device, C.byref(desc), x, weight, bias, y, stats[0], stats[1], ws, size)
    return y, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        w, b = (t if t is None else t.detach().contiguous() for t in (weight, bias))
        v = _rows_view(x.detach())
        y, stats = _forward(v, groups, w, b, eps, act)
        ctx.save_for_backward(v, w, b, stats)
        ctx.groups, ctx.eps, ctx.act, ctx.shape = groups, eps, act, x.shape
        return y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, b, stats = ctx.saved_tensors
        d = _rows_view(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dw = torch.empty_like(w) if w is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(b) if b is not None and ctx.needs_input_grad[2] else None
        desc = _desc(x, ctx.groups, ctx.eps, ctx.act, w if w is not None else b, d)
        ws, size = _workspace(desc, True, x.device)
        _lib.call("ps_group_norm_backward", x.device, C.byref(desc), x, d, w, b, stats[0], stats[1], dx, dw, db, ws,
                  size)
        return dx.view(ctx.shape), dw, db, None, None, None


def group_norm(x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, activation: str = "none") -> Tensor:
    """act(group_norm(x) * weight + bias) for a channels-last x [n, ..., c] on the GPU, one fused pass each way.

    The statistics of a (sample, group) are over all positions and its c / num_groups channels (biased variance), as
    torch.nn.functional.group_norm has them for channels-first tensors.  x: fp32, bf16 or fp16, any strides (a view
    [n, positions, c] with unit channel stride is read in place, anything else is copied first).  weight, bias [c]: x's
    type or fp32, each optional, both of one type.  activation: none, relu, silu, gelu (exact) or sigmoid.  The result
    is contiguous.  Differentiable once in x, weight and bias; results repeat bit for bit."""
    _lib.check_tensors("group_norm", x, weight=weight, bias=bias)
    act = _lib.activation_code("group_norm", activation)
    if x.dim() < 2:
        raise ValueError(f"group_norm: x is [n, ..., channels], got {tuple(x.shape)}")
    c = x.shape[-1]
    if num_groups < 1 or c == 0 or c % num_groups:
        raise ValueError(f"group_norm: {c} channels do not divide into {num_groups} groups")
    if not eps >= 0:
        raise ValueError(f"group_norm: eps {eps} is negative")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (c,) or t.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f"group_norm: {name} is [{c}] in {x.dtype} or float32, got {tuple(t.shape)} {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("group_norm: weight and bias have different types")
    if x.numel() == 0:       # no statistics, no elements: gradients of the parameters are zero
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        tied = [t.sum() * 0 for t in (x, weight, bias) if t is not None and t.requires_grad]
        return y + sum(tied).to(x.dtype) if tied and torch.is_grad_enabled() else y
    if _lib.wants_grad(x, weight, bias):
        return _GroupNorm.apply(x, weight, bias, num_groups, float(eps), act)
    w, b = (t if t is None else t.detach().contiguous() for t in (weight, bias))
    return _forward(_rows_view(x.detach()), num_groups, w, b, float(eps), act)[0].view(x.shape)


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm (same parameters, same state) followed by an activation, on images [n, c, h, w] kept in
    torch.channels_last: the kernel reads and writes that memory as it lies (other layouts are copied to it)."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "none", device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        _lib.activation_code("GroupNormAct", activation)
        self.activation = activation

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() < 3 or x.shape[1] != self.num_channels:
            raise ValueError(f"GroupNormAct: x is [n, {self.num_channels}, ...], got {tuple(x.shape)}")
        y = group_norm(x.movedim(1, -1), self.num_groups, self.weight, self.bias, self.eps, self.activation)
        return y.movedim(-1, 1)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
