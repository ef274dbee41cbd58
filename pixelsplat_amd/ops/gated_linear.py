"""Gated projection of a feed-forward block (csrc/gated_linear.hip)."""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _lib


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor] = None,
                 b_up: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up) in one kernel: [..., dim] -> [..., hidden].

    x [..., dim] fp32, bf16 or fp16 on the GPU; weights [hidden, dim] and biases [hidden] (each optional) in its type.
    activation: silu, gelu (exact), relu, sigmoid or none.  Any number of rows, one included; x and the weights are
    read in place when their rows are 16-byte aligned (dim a multiple of 8, or 4 in fp32), and copied otherwise.
    fp32 products are fp32 throughout; 16-bit ones accumulate in fp32 and round once.  The 16-bit backward also rounds the
    gradients of the two projections, which its products read (in fp16 within a range of their own: it neither overflows nor
    loses small gradients there).  Differentiable once in all five
    tensors: fp32 keeps both projections for it (8 bytes a hidden value), 16-bit types keep only their inputs.
    Under torch.autocast all five take its type, as in torch's own products.  Results repeat bit for bit."""
    act = _lib.activation_code("gated_linear", activation)
    return _lib.binding().gated_linear(x, w_gate, w_up, b_gate, b_up, act)
