"""Gated projection of a feed-forward block (csrc/gated_linear.hip)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch import Tensor

from . import _lib

GATES = ("relu", "silu", "gelu", "sigmoid", "none")


def _chunked(t: Tensor, pad: int) -> Tensor:
    """[rows, dim] as the kernels read it: unit column stride, rows of whole 16-byte chunks that start on one.  Read in
    place where it lies like that, copied (with `pad` zero columns) otherwise."""
    vec = 16 // t.element_size()
    if pad:
        return torch.nn.functional.pad(t, (0, pad))
    if t.shape[1] > 1 and t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % vec or t.stride(0) < t.shape[1])) \
            or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _desc(x: Tensor, w: Tensor, act: int, dh: Optional[Tensor] = None) -> _lib.PsGatedLinearDesc:
    return _lib.PsGatedLinearDesc(x.shape[0], x.shape[1], w.shape[0], _lib.DTYPES[x.dtype], act, 0, _stride(x),
                                  _stride(w), _stride(dh) if dh is not None else 0)


def _operands(x2: Tensor, wg: Tensor, wu: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    pad = -x2.shape[1] % (16 // x2.element_size())
    x2, wg, wu = (_chunked(t, pad) for t in (x2, wg, wu))
    if _stride(wg) != _stride(wu):           # one row stride for both
        wg, wu = (t.clone(memory_format=torch.contiguous_format) for t in (wg, wu))
    return x2, wg, wu


def _forward(x2, wg, wu, bg, bu, act: int, keep: bool):
    h = torch.empty((x2.shape[0], wg.shape[0]), dtype=x2.dtype, device=x2.device)
    kept = torch.empty((2, *h.shape), dtype=torch.float32, device=x2.device) if keep else None
    desc = _desc(x2, wg, act)
    _lib.call("ps_gated_linear_forward", x2.device, C.byref(desc), x2, wg, wu, bg, bu, h,
              kept[0] if keep else None, kept[1] if keep else None)
    return h, kept


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        x2, wg, wu = _operands(x.detach().reshape(-1, x.shape[-1]), w_gate.detach(), w_up.detach())
        bg, bu = (b if b is None else b.detach().contiguous() for b in (b_gate, b_up))
        h, kept = _forward(x2, wg, wu, bg, bu, act, x.dtype == torch.float32)
        ctx.save_for_backward(x2, wg, wu, bg, bu, kept)
        ctx.act, ctx.shape = act, x.shape
        return h.view(*x.shape[:-1], h.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x2, wg, wu, bg, bu, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        d2 = dh.reshape(x2.shape[0], wg.shape[0])
        if (d2.shape[1] > 1 and d2.stride(1) != 1) or (d2.shape[0] > 1 and d2.stride(0) < d2.shape[1]):
            d2 = d2.contiguous()
        new = lambda t, want: torch.empty(t.shape, dtype=t.dtype, device=t.device) if want else None  # noqa: E731
        dx, dwg, dwu = new(x2, need[0]), new(wg, need[1]), new(wu, need[2])
        dbg = new(bg, need[3]) if bg is not None else None
        dbu = new(bu, need[4]) if bu is not None else None
        desc = _desc(x2, wg, ctx.act, d2)
        size = _lib.load().ps_gated_linear_backward_workspace_bytes(C.byref(desc))
        ws = torch.empty((size,), dtype=torch.uint8, device=x2.device)
        _lib.call("ps_gated_linear_backward", x2.device, C.byref(desc), x2, wg, wu, bg, bu,
                  kept[0] if kept is not None else None, kept[1] if kept is not None else None, d2, dx, dwg, dwu, dbg,
                  dbu, ws, size)
        dim = ctx.shape[-1]
        cut = lambda t: t if t is None or t.shape[1] == dim else t[:, :dim]  # noqa: E731
        dx = None if dx is None else cut(dx).reshape(ctx.shape)
        return dx, cut(dwg), cut(dwu), dbg, dbu, None


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor] = None,
                 b_up: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up) in one kernel: [..., dim] -> [..., hidden].

    x [..., dim] fp32, bf16 or fp16 on the GPU; weights [hidden, dim] and biases [hidden] (each optional) in its type.
    activation: silu, gelu (exact), relu, sigmoid or none.  Any number of rows, one included; x and the weights are
    read in place when their rows are 16-byte aligned (dim a multiple of 8, or 4 in fp32), and copied otherwise.
    fp32 products are fp32 throughout; 16-bit ones accumulate in fp32 and round once.  Differentiable once in all five
    tensors: fp32 keeps both projections for it (8 bytes a hidden value), 16-bit types keep only their inputs.
    Results repeat bit for bit."""
    _lib.check_tensors("gated_linear", x, w_gate=w_gate, w_up=w_up, b_gate=b_gate, b_up=b_up)
    act = _lib.activation_code("gated_linear", activation, GATES)
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1]:
        raise ValueError(f"gated_linear: x [..., dim] and two weights [hidden, dim], got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    hidden, dim = w_gate.shape
    for name, t, shape in (("w_gate", w_gate, w_gate.shape), ("w_up", w_up, w_gate.shape),
                           ("b_gate", b_gate, (hidden,)), ("b_up", b_up, (hidden,))):
        if t is not None and (t.dtype != x.dtype or tuple(t.shape) != tuple(shape)):
            raise ValueError(f"gated_linear: {name} is {tuple(shape)} in {x.dtype}, got {tuple(t.shape)} {t.dtype}")
    if hidden == 0 or dim == 0 or x.numel() == 0:
        if dim == 0:
            raise ValueError("gated_linear: dim is 0")
        y = x.new_zeros((*x.shape[:-1], hidden))
        tied = [t.sum() * 0 for t in (x, w_gate, w_up, b_gate, b_up) if t is not None and t.requires_grad]
        return y + sum(tied) if tied and torch.is_grad_enabled() else y
    if _lib.wants_grad(x, w_gate, w_up, b_gate, b_up):
        return _GatedLinear.apply(x, w_gate, w_up, b_gate, b_up, act)
    x2, wg, wu = _operands(x.detach().reshape(-1, dim), w_gate.detach(), w_up.detach())
    bg, bu = (b if b is None else b.detach().contiguous() for b in (b_gate, b_up))
    return _forward(x2, wg, wu, bg, bu, act, False)[0].view(*x.shape[:-1], hidden)
