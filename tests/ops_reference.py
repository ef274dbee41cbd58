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
