"""Attention / PreNorm / FeedForward / Transformer with the reference's parameter names and
call conventions (src/model/transformer/{attention,pre_norm,feed_forward,transformer}.py,
vendored there from stelzner/srt).  Plain PyTorch: the dense projections are library GEMMs; the
epipolar cross-attention is routed to the fused HIP kernel by EpipolarTransformer.

Beyond the reference, off by default: `relative_buckets` gives self-attention over a token grid a
learned relative position bias (ops.relative_attention), and GatedFeedForward is a feed-forward
layer with a gated projection (ops.gated_linear)."""
from __future__ import annotations

import torch
from torch import nn
from torch.nn.modules import module as nn_module

from ..ops import RelativePositionBias, gated_linear


class FeedForward(nn.Module):
    def __init__(self, dim, hidden_dim, dropout=0.0):
        super().__init__()
        self.net = nn.Sequential(nn.Linear(dim, hidden_dim), nn.GELU(), nn.Dropout(dropout),
                                 nn.Linear(hidden_dim, dim), nn.Dropout(dropout))

    def forward(self, x):
        return self.net(x)


class GatedFeedForward(nn.Module):
    """FeedForward with a gated projection: down(act(x w_gate^T + b_gate) * (x w_up^T + b_up)), the
    bracket one kernel (ops.gated_linear: no projection reaches memory in 16-bit types)."""

    def __init__(self, dim, hidden_dim, dropout=0.0, activation="silu", bias=True):
        super().__init__()
        self.activation = activation
        self.gate = nn.Linear(dim, hidden_dim, bias=bias)
        self.up = nn.Linear(dim, hidden_dim, bias=bias)
        self.down = nn.Linear(hidden_dim, dim, bias=bias)
        self.dropout = nn.Dropout(dropout)

    def forward(self, x):
        h = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, self.activation)
        return self.dropout(self.down(self.dropout(h)))


class PreNorm(nn.Module):
    def __init__(self, dim, fn):
        super().__init__()
        self.norm = nn.LayerNorm(dim)
        self.fn = fn

    def forward(self, x, **kwargs):
        return self.fn(self.norm(x), **kwargs)


def _hooked(module: nn.Module) -> bool:
    """Whether a hook of any kind waits for a call of `module`, one on all modules included."""
    return any(len(hooks) > 0 for owner, prefix in ((module, ""), (nn_module, "_global"))
               for hooks in (getattr(owner, prefix + kind) for kind in (
                   "_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")))


class Attention(nn.Module):
    """relative_buckets > 0 (self-attention only): a learned bias on the tokens' offsets on a grid,
    relative_buckets logarithmic buckets an axis.  forward then takes the grid (rows, columns) of the
    tokens, and a key mask [batch, tokens] for padded batches."""

    def __init__(self, dim, heads=8, dim_head=64, dropout=0.0, selfatt=True, kv_dim=None,
                 relative_buckets=0):
        super().__init__()
        inner_dim = dim_head * heads
        project_out = not (heads == 1 and dim_head == dim)
        self.heads = heads
        self.scale = dim_head ** -0.5
        self.attend = nn.Softmax(dim=-1)   # visualisers hook this module
        if selfatt:
            self.to_qkv = nn.Linear(dim, inner_dim * 3, bias=False)
        else:
            self.to_q = nn.Linear(dim, inner_dim, bias=False)
            self.to_kv = nn.Linear(kv_dim, inner_dim * 2, bias=False)
        if relative_buckets and not selfatt:
            raise ValueError("a relative position bias needs self-attention: keys on the queries' grid")
        self.relative_bias = RelativePositionBias(heads, relative_buckets) if relative_buckets else None
        self.to_out = (nn.Sequential(nn.Linear(inner_dim, dim), nn.Dropout(dropout))
                       if project_out else nn.Identity())

    def forward(self, x, z=None, grid=None, key_mask=None):
        if (grid is None) != (self.relative_bias is None) or (key_mask is not None and grid is None):
            raise ValueError("a grid (and with it a key mask) goes with relative_buckets, and only with it")
        if z is None:
            q, k, v = self.to_qkv(x).chunk(3, dim=-1)
        else:
            q = self.to_q(x)
            k, v = self.to_kv(z).chunk(2, dim=-1)
        split = lambda t: t.reshape(t.shape[0], t.shape[1], self.heads, -1).transpose(1, 2)
        q, k, v = split(q), split(k), split(v)
        if self.relative_bias is not None and not _hooked(self.attend):
            out = self.relative_bias(q, k, v, grid, key_mask, self.scale).transpose(1, 2)
        else:   # a hook on `attend` sees the logits, the attention weights or their gradients
            logits = torch.matmul(q, k.transpose(-1, -2)) * self.scale
            if grid is not None:
                logits = logits + self.relative_bias.matrix(grid).to(logits.dtype)
            if key_mask is not None:
                logits = logits.masked_fill(~key_mask[:, None, None], float("-inf"))
            attn = self.attend(logits)
            if key_mask is not None:      # rows without keys
                attn = torch.where(key_mask.any(1)[:, None, None, None], attn, torch.zeros_like(attn))
                v = torch.where(key_mask[:, None, :, None], v, torch.zeros_like(v))
            out = torch.matmul(attn, v).transpose(1, 2)
        return self.to_out(out.reshape(out.shape[0], out.shape[1], -1))


class Transformer(nn.Module):
    def __init__(self, dim, depth, heads, dim_head, mlp_dim, dropout=0.0, selfatt=True,
                 kv_dim=None, feed_forward_layer=FeedForward, relative_buckets=0):
        super().__init__()
        self.layers = nn.ModuleList([])
        for _ in range(depth):
            self.layers.append(nn.ModuleList([
                PreNorm(dim, Attention(dim, heads=heads, dim_head=dim_head, dropout=dropout,
                                       selfatt=selfatt, kv_dim=kv_dim,
                                       relative_buckets=relative_buckets)),
                PreNorm(dim, feed_forward_layer(dim, mlp_dim, dropout=dropout)),
            ]))

    def forward(self, x, z=None, grid=None, key_mask=None, **kwargs):
        for attn, ff in self.layers:
            x = attn(x, z=z, grid=grid, key_mask=key_mask) + x
            x = ff(x, **kwargs) + x
        return x
