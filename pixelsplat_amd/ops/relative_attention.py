"""Attention over a token grid with a learned relative position bias (csrc/relative_attention.hip)."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch
from torch import Tensor, nn

from . import _lib

_STRIDES = C.c_int64 * 3


def relative_buckets(grid: tuple[int, int], buckets_per_axis: int = 32, max_distance: int = 128,
                     device=None) -> Tensor:
    """[2 gh - 1, 2 gw - 1] int32 for `relative_attention`: the bucket of a (row, column) offset key - query on a grid of
    gh x gw tokens.  Each axis has buckets_per_axis buckets, half of them for offsets > 0: one for every distance below
    buckets_per_axis / 4, then logarithmically wider ones that reach max_distance, the last holding all that is
    farther.  The two axes' buckets are combined row-major; an axis of one token has one bucket, so a 1 x n grid is a
    sequence with buckets_per_axis buckets.  The number of buckets is relative_bucket_count(grid, buckets_per_axis)."""
    gh, gw = _grid(grid)
    columns = 1 if gw == 1 else buckets_per_axis
    rows, cols = (_axis(n, buckets_per_axis, max_distance) for n in (gh, gw))
    return (rows[:, None] * columns + cols[None]).int().to(device)


def _axis(n: int, buckets: int, max_distance: int) -> Tensor:
    half, exact = buckets // 2, buckets // 4
    if buckets < 4 or buckets % 4 or max_distance <= exact:
        raise ValueError(f"relative_buckets: buckets_per_axis {buckets} is a multiple of 4 and max_distance "
                         f"{max_distance} above a quarter of it")
    d = torch.arange(-(n - 1), n, dtype=torch.float64)
    steps = torch.log(d.abs().clamp(min=1) / exact) / math.log(max_distance / exact) * (half - exact)
    far = (exact + steps.floor()).clamp(max=half - 1)
    return (torch.where(d.abs() < exact, d.abs(), far) + half * (d > 0)).long()


def relative_bucket_count(grid: tuple[int, int], buckets_per_axis: int = 32) -> int:
    gh, gw = _grid(grid)
    return (1 if gh == 1 else buckets_per_axis) * (1 if gw == 1 else buckets_per_axis)


def _grid(grid) -> tuple[int, int]:
    gh, gw = grid
    if gh < 1 or gw < 1:
        raise ValueError(f"a grid has at least one row and one column, got {tuple(grid)}")
    return gh, gw


def _rows(t: Tensor, pad: int) -> Tensor:
    """[batch, heads, tokens, dim] as the kernels read it: rows that start on 16 bytes, at positive strides."""
    if pad:
        return torch.nn.functional.pad(t, (0, pad))
    vec = 16 // t.element_size()
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and t.stride(2) < 1 << 24
    if not ok or any(t.shape[i] > 1 and t.stride(i) % vec for i in range(3)):
        # copied token-major, as a packed projection would lay it out
        return t.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)
    return t


def _strides(t: Tensor):
    vec = 16 // t.element_size()
    return _STRIDES(*(t.stride(i) if t.shape[i] > 1 else vec for i in range(3)))


def _desc(q, k, v, table, buckets, scale, start, mask, dout=None) -> _lib.PsRelativeAttentionDesc:
    gh, gw = (buckets.shape[0] + 1) // 2, (buckets.shape[1] + 1) // 2
    return _lib.PsRelativeAttentionDesc(
        q.shape[0], q.shape[1], q.shape[2], start, gh, gw, q.shape[3], _lib.DTYPES[q.dtype], table.shape[0],
        int(table.dtype == torch.float32), scale, 0, _strides(q), _strides(k), _strides(v),
        _strides(dout) if dout is not None else _STRIDES(), mask.stride(0) if mask is not None else 0)


def _new(like: Tensor) -> Tensor:
    """[batch, heads, tokens, dim], token-major in memory: merging the heads is a view"""
    b, h, n, d = like.shape
    return torch.empty((b, n, h, d), dtype=like.dtype, device=like.device).transpose(1, 2)


def _forward(q, k, v, table, buckets, mask, scale, start, keep: bool):
    device, (b, h, n, _) = q.device, q.shape
    desc = _desc(q, k, v, table, buckets, scale, start, mask)
    size = _lib.load().ps_relative_attention_workspace_bytes(C.byref(desc), 0)
    if size == 0:
        raise RuntimeError("relative_attention: unsupported configuration (see its limits)")
    out = _new(q)
    bias = torch.empty((h, buckets.numel()), dtype=torch.float32, device=device)
    stats = torch.empty((2, b, h, (n + 63) // 64 * 64), dtype=torch.float32, device=device) if keep else None
    out32 = torch.empty((b, n, h, q.shape[3]), dtype=torch.float32, device=device) \
        if keep and q.dtype != torch.float32 else None
    ws = torch.empty((size,), dtype=torch.uint8, device=device)
    _lib.call("ps_relative_attention_forward", device, C.byref(desc), q, k, v, mask, buckets, table, out, out32, stats,
              bias, ws, size)
    return out, (out32 if out32 is not None else out), stats, bias


class _RelativeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, mask, scale, start):
        dim = q.shape[3]
        pad = -dim % (16 // q.element_size())
        q, k, v = (_rows(t.detach(), pad) for t in (q, k, v))
        t = table.detach().contiguous()
        out, kept, stats, bias = _forward(q, k, v, t, buckets, mask, scale, start, True)
        ctx.save_for_backward(q, k, v, t, buckets, mask, kept, stats, bias)
        ctx.args, ctx.dim = (scale, start), dim
        return out[..., :dim] if pad else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, table, buckets, mask, kept, stats, bias = ctx.saved_tensors
        scale, start = ctx.args
        dout = _rows(dout, q.shape[3] - ctx.dim)
        need = ctx.needs_input_grad
        dq, dk, dv = (_new(t) if want else None for t, want in zip((q, k, v), need))
        dtable = torch.empty_like(table) if need[3] else None
        desc = _desc(q, k, v, table, buckets, scale, start, mask, dout)
        size = _lib.load().ps_relative_attention_workspace_bytes(C.byref(desc), 1)
        ws = torch.empty((size,), dtype=torch.uint8, device=q.device)
        _lib.call("ps_relative_attention_backward", q.device, C.byref(desc), q, k, v, mask, buckets, bias, kept, stats,
                  dout, dq, dk, dv, dtable, ws, size)
        if q.shape[3] != ctx.dim:
            dq, dk, dv = (t if t is None else t[..., :ctx.dim] for t in (dq, dk, dv))
        return dq, dk, dv, dtable, None, None, None, None


def relative_attention(q: Tensor, k: Tensor, v: Tensor, table: Tensor, buckets: Tensor,
                       key_mask: Optional[Tensor] = None, scale: Optional[float] = None,
                       query_start: int = 0) -> Tensor:
    """softmax(scale q k^T + bias) v over a grid of gh x gw tokens, bias[head, i, j] = table[bucket(j - i), head].

    q [batch, heads, queries, dim]; k, v [batch, heads, gh gw, dim], tokens numbered by rows: fp32, bf16 or fp16 on the
    GPU, any strides (views of a packed projection are read in place; rows that do not start on 16 bytes are copied).
    The queries are the tokens query_start, query_start + 1, ...: all of them, a block, or a single one.
    table [n, heads] in q's type or fp32; buckets [2 gh - 1, 2 gw - 1] int32 (relative_buckets, or any map of offsets;
    its shape names the grid; an entry outside 0 .. n - 1 is an offset without bias).  key_mask [batch, gh gw] bool,
    True for a key that is there; the values of masked keys do not matter, NaN included, and a row without keys is
    zero.  scale: dim ** -0.5 by default.  Returns [batch, heads, queries, dim], token-major in memory.

    dim <= 128, at most 2^20 keys, gw <= 512 on grids of more than one row.  Differentiable once in q, k, v and table;
    the gradient of the table is summed over the batch.  16-bit types accumulate in fp32 and round probabilities for
    their product with v.  Results repeat bit for bit."""
    _lib.check_tensors("relative_attention", q, k=k, v=v, table=table, buckets=buckets, key_mask=key_mask)
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError("relative_attention: q [batch, heads, queries, dim], k and v [batch, heads, keys, dim], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype or table.dtype not in (q.dtype, torch.float32):
        raise ValueError(f"relative_attention: k and v are {q.dtype} as q, the table that or float32, got {k.dtype}, "
                         f"{v.dtype}, {table.dtype}")
    if buckets.dtype != torch.int32 or buckets.dim() != 2 or buckets.shape[0] % 2 == 0 or buckets.shape[1] % 2 == 0:
        raise ValueError("relative_attention: buckets is [2 rows - 1, 2 columns - 1] int32, got "
                         f"{tuple(buckets.shape)} {buckets.dtype}")
    b, h, n, dim = q.shape
    gh, gw = (buckets.shape[0] + 1) // 2, (buckets.shape[1] + 1) // 2
    if k.shape[2] != gh * gw:
        raise ValueError(f"relative_attention: {k.shape[2]} keys on a grid of {gh} x {gw}")
    if query_start < 0 or query_start + n > gh * gw:
        raise ValueError(f"relative_attention: queries {query_start} .. {query_start + n - 1} of {gh * gw} tokens")
    if table.dim() != 2 or table.shape[1] != h or table.shape[0] == 0:
        raise ValueError(f"relative_attention: table is [buckets, {h}], got {tuple(table.shape)}")
    if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, gh * gw)):
        raise ValueError(f"relative_attention: key_mask is [{b}, {gh * gw}] bool, got {tuple(key_mask.shape)} "
                         f"{key_mask.dtype}")
    if not 0 < dim <= 128 or gh * gw > 1 << 20 or (gh > 1 and gw > 512):
        raise ValueError(f"relative_attention: dim {dim} is 1 .. 128, a grid of {gh} x {gw} has at most 2^20 tokens and "
                         "512 columns (one row: any)")
    scale = dim ** -0.5 if scale is None else float(scale)
    if q.numel() == 0:
        y = torch.zeros_like(q, memory_format=torch.contiguous_format)
        tied = [t.sum() * 0 for t in (q, k, v, table) if t.requires_grad]
        return y + sum(tied).to(q.dtype) if tied and torch.is_grad_enabled() else y
    buckets = buckets.contiguous()
    if key_mask is not None and key_mask.stride(1) != 1:
        key_mask = key_mask.contiguous()
    if _lib.wants_grad(q, k, v, table):
        return _RelativeAttention.apply(q, k, v, table, buckets, key_mask, scale, query_start)
    pad = -dim % (16 // q.element_size())
    q, k, v = (_rows(t.detach(), pad) for t in (q, k, v))
    out = _forward(q, k, v, table.detach().contiguous(), buckets, key_mask, scale, query_start, False)[0]
    return out[..., :dim] if pad else out


class RelativePositionBias(nn.Module):
    """The learned table of a relative position bias for `heads` heads: buckets_per_axis logarithmic buckets a grid axis
    (relative_buckets).  One table of buckets_per_axis^2 rows serves grids of every size; the bucket map of a grid is
    made when it is first used and kept with the module."""

    def __init__(self, heads: int, buckets_per_axis: int = 32, max_distance: int = 128):
        super().__init__()
        _axis(1, buckets_per_axis, max_distance)          # checks the arguments
        self.buckets_per_axis, self.max_distance = buckets_per_axis, max_distance
        self.table = nn.Parameter(torch.zeros(buckets_per_axis ** 2, heads))
        self._maps: dict = {}

    def buckets(self, grid: tuple[int, int], device) -> Tensor:
        key = (*grid, torch.device(device))
        if key not in self._maps:
            rows, cols = (_axis(n, self.buckets_per_axis, self.max_distance) for n in _grid(grid))
            self._maps[key] = (rows[:, None] * self.buckets_per_axis + cols[None]).int().to(device)
        return self._maps[key]

    def forward(self, q: Tensor, k: Tensor, v: Tensor, grid: tuple[int, int], key_mask: Optional[Tensor] = None,
                scale: Optional[float] = None, query_start: int = 0) -> Tensor:
        return relative_attention(q, k, v, self.table, self.buckets(grid, q.device), key_mask, scale, query_start)
