"""Plain 64-bit implementations of the image-transformer operators, for their tests."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # finfo.eps / 2
U = 2.0 ** -24            # a rounding of fp32 arithmetic
# smallest steps of the types: what a rounded value may be off by where it is subnormal
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    assert name == "sigmoid"
    return torch.sigmoid(z)


def group_norm(x, groups, weight, bias, eps, activation):
    n, c = x.shape[0], x.shape[-1]
    t = x.reshape(n, -1, groups, c // groups)
    mean = t.mean((1, 3), keepdim=True)
    var = (t - mean).square().mean((1, 3), keepdim=True)
    z = ((t - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    z = z if weight is None else z * weight
    z = z if bias is None else z + bias
    return act(activation, z)


def within(got, want, bound, what):
    """Every element of `got` is within `bound` (a tensor or a number) of `want`."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert (over <= 0).all(), (f"{what}: element {at}: {got.flatten()[at].item():.9g} for {want.flatten()[at].item():.9g}, "
                               f"{over.flatten()[at].item():.3g} over the bound")


def slope(name, z):
    """act'(z), and a bound of |act''| (relu: its jump is the caller's)"""
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    s = torch.sigmoid(z)
    if name == "silu":
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return s * (1 - s)


def gated_linear(x, wg, wu, bg, bu, activation, dh=None):
    """h, and with dh the gradients and what their bounds need (formulas, 64 bits)"""
    a, u = x @ wg.T, x @ wu.T
    a = a if bg is None else a + bg
    u = u if bu is None else u + bu
    value = act(activation, a)
    if dh is None:
        return value * u
    du, da = dh * value, dh * u * slope(activation, a)
    return value * u, dict(x=da @ wg + du @ wu, w_gate=da.T @ x, w_up=du.T @ x, b_gate=da.sum(0), b_up=du.sum(0)), \
        dict(a=a, u=u, value=value, da=da, du=du)


def grid_offsets(grid, start, queries, device):
    """[queries, keys] index into a flattened [2 gh - 1, 2 gw - 1] map"""
    gh, gw = grid
    at = torch.arange(gh * gw, device=device)
    y, x = at // gw, at % gw
    mine = slice(start, start + queries)
    return (y[None] - y[mine, None] + gh - 1) * (2 * gw - 1) + x[None] - x[mine, None] + gw - 1


def relative_attention(q, k, v, table, buckets, mask, scale, start, do=None):
    """out and, with do, (dq, dk, dv, dtable); and what their bounds need (formulas, 64 bits)"""
    grid = (buckets.shape[0] + 1) // 2, (buckets.shape[1] + 1) // 2
    bucket = buckets.reshape(-1).long()[grid_offsets(grid, start, q.shape[2], q.device)]
    there = (bucket >= 0) & (bucket < table.shape[0])
    bias = torch.where(there[..., None], table[bucket.clamp(0, table.shape[0] - 1)], torch.zeros((), dtype=q.dtype, device=q.device))
    bias = bias.permute(2, 0, 1)[None]
    if mask is not None:          # what a masked key holds does not matter
        k, v = (torch.where(mask[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    s = scale * (q @ k.transpose(-1, -2)) + bias
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(e), e / total)
    out = p @ v
    if do is None:
        return out, dict(p=p, bias=bias, bucket=bucket, there=there, k=k, v=v)
    dp = do @ v.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dtable = torch.zeros_like(table)
    flat = torch.where(there, bucket, torch.full_like(bucket, table.shape[0])).reshape(-1)
    grow = torch.zeros((table.shape[0] + 1, table.shape[1]), dtype=table.dtype, device=table.device)
    grow.index_add_(0, flat, ds.sum(0).flatten(1).T)
    dtable = grow[:-1]
    return out, (scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q), p.transpose(-1, -2) @ do, dtable), \
        dict(p=p, bias=bias, flat=flat, ds=ds, dp=dp, delta=delta, k=k, v=v)
