"""Group norm with an activation on channels-last maps (csrc/group_norm.hip)."""
from __future__ import annotations

from typing import Optional

from torch import Tensor, nn

from . import _lib


def group_norm(x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, activation: str = "none") -> Tensor:
    """act(group_norm(x) * weight + bias) for a channels-last x [n, ..., c] on the GPU, one fused pass each way.

    The statistics of a (sample, group) are over all positions and its c / num_groups channels (biased variance), as
    torch.nn.functional.group_norm has them for channels-first tensors.  x: fp32, bf16 or fp16, any strides (a view
    [n, positions, c] with unit channel stride is read in place, anything else is copied first).  weight, bias [c]: x's
    type or fp32, each optional, both of one type.  activation: none, relu, silu, gelu (exact) or sigmoid.  The result
    is contiguous, in x's type under torch.autocast too.  Differentiable once in x, weight and bias; results repeat bit for bit."""
    act = _lib.activation_code("group_norm", activation)
    return _lib.binding().group_norm(x, num_groups, weight, bias, eps, act)


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
