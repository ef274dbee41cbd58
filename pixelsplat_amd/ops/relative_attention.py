"""Attention over a token grid with a learned relative position bias (csrc/relative_attention.hip)."""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor, nn

from . import _lib

def relative_buckets(grid: tuple[int, int], buckets_per_axis: int = 32, max_distance: int = 128,
                     device=None) -> Tensor:
    """[2 gh - 1, 2 gw - 1] int32 for `relative_attention`: the bucket of a (row, column) offset key - query on a grid of
    gh x gw tokens.  Each axis has buckets_per_axis buckets, half of them for offsets > 0: one for every distance below
    buckets_per_axis / 4, then logarithmically wider ones that reach max_distance, the last holding all that is
    farther.  The two axes' buckets are combined row-major; an axis of one token has one bucket, so a 1 x n grid is a
    sequence with buckets_per_axis buckets.  The number of buckets is relative_bucket_count(grid, buckets_per_axis)."""
    columns = 1 if _grid(grid)[1] == 1 else buckets_per_axis
    return _map(grid, buckets_per_axis, max_distance, columns, device)


def _map(grid: tuple[int, int], buckets: int, max_distance: int, columns: int, device) -> Tensor:
    # an ordinary tensor also where it is asked for in inference mode: training saves it for its backward pass
    with torch.inference_mode(False):
        rows, cols = (_axis(n, buckets, max_distance) for n in _grid(grid))
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
    zero.  scale: dim ** -0.5 by default.  Returns [batch, heads, queries, dim], token-major in memory; it may be changed
    in place (in fp32 not before its backward pass, which reads it).

    Under torch.autocast q, k and v take its type, as in torch's own products; the table keeps its own.

    dim <= 128, at most 2^20 keys, gw <= 512 on grids of more than one row.  The table's gradient takes a workspace of
    queries x keys / 8 bytes a head, twice that on grids of more than one row, and reads the map once a bucket unless
    neighbouring offsets' buckets are near each other.  Differentiable once in q, k, v and table;
    the gradient of the table is summed over the batch.  16-bit types accumulate in fp32; the backward rounds probabilities
    and the logits' gradients to them for its products (in fp16 within a range of their own: they neither overflow nor lose
    small values there).  Results repeat bit for bit."""
    return _lib.binding().relative_attention(q, k, v, table, buckets, key_mask, scale, query_start)


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
            self._maps[key] = _map(grid, self.buckets_per_axis, self.max_distance, self.buckets_per_axis, device)
        return self._maps[key]

    def matrix(self, grid: tuple[int, int]) -> Tensor:
        """[heads, tokens, tokens]: the bias written out, for what has to see the attention weights."""
        gh, gw = _grid(grid)
        at = torch.arange(gh * gw, device=self.table.device)
        rows, cols = (at // gw)[None] - (at // gw)[:, None], (at % gw)[None] - (at % gw)[:, None]
        return self.table[self.buckets(grid, self.table.device).long()[rows + gh - 1, cols + gw - 1]].permute(2, 0, 1)

    def forward(self, q: Tensor, k: Tensor, v: Tensor, grid: tuple[int, int], key_mask: Optional[Tensor] = None,
                scale: Optional[float] = None, query_start: int = 0) -> Tensor:
        return relative_attention(q, k, v, self.table, self.buckets(grid, q.device), key_mask, scale, query_start)
