"""The activations of the image-transformer operators at every 16-bit number: value and slope, through gated_linear.

A unit of weight 1 on one of eight inputs and an up projection of 1 (its bias) leave h = act(z) and dx = act'(z), each
rounded once.  Bounds: half a step of the value; GELU's tail is off by 2^-14 of itself, exp(-z^2 / 2) by (z^2 + 8) 2^-24 of
itself (the argument's rounding), cdf of z > 0 by 2.5e-7; the slope is the sum cdf + z bell / sqrt(2 pi), with 4 roundings
more.  Sigmoids are off by (2 |z| + 8) 2^-24 of themselves (the exponential's argument and base), their slope by twice that;
silu's slope s (1 + z (1 - s)) by that of s, and s times the errors of its sum.  fp32 numbers below 2^-126 may be zero."""
import math

import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu


def numbers(dtype, limit, dev):
    z = torch.arange(-1 << 15, 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    return z[z.isfinite() & (z.abs() <= limit)].to(dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_gelu_at_every_number(gpu_device, dtype):
    from pixelsplat_amd.ops import gated_linear

    z = numbers(dtype, 200.0, gpu_device)
    x = torch.zeros((len(z), 8), dtype=dtype, device=gpu_device)
    x[:, 0] = z
    x.requires_grad_()
    w = torch.zeros((1, 8), dtype=dtype, device=gpu_device)
    w[0, 0] = 1
    one = torch.ones(1, dtype=dtype, device=gpu_device)
    h = gated_linear(x, w, torch.zeros_like(w), None, one, "gelu")
    dx = torch.autograd.grad(h, x, torch.ones_like(h))[0][:, 0]
    zd = z.double()
    cdf, bell = 0.5 * torch.erfc(-zd / math.sqrt(2)), torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    e_bell = bell * (zd * zd + 8) * R.U + 2.0 ** -126
    e_cdf = torch.where(zd < 0, cdf * (2.0 ** -14 + (zd * zd + 8) * R.U) + 2.0 ** -126, 2.5e-7 * torch.ones_like(cdf))
    value, slope = zd * cdf, cdf + zd * bell
    half, tiny = R.HALF_STEP[dtype], R.TINY[dtype]
    R.within(h[:, 0], value, half * value.abs() + 1.01 * zd.abs() * (e_cdf + 4 * R.U * cdf) + tiny, "gelu")
    # da passes through fp16's own range there, and once more through rounding, of what is representable
    R.within(dx, slope, half * slope.abs() + 1.01 * (e_cdf + zd.abs() * e_bell + 4 * R.U * (cdf + (zd * bell).abs())) + tiny,
             "gelu's slope")


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_sigmoids_at_every_number(gpu_device, dtype, act):
    from pixelsplat_amd.ops import gated_linear

    z = numbers(torch.bfloat16 if dtype == torch.float32 else dtype, 200.0, gpu_device).to(dtype)
    x = torch.zeros((len(z), 8), dtype=dtype, device=gpu_device)
    x[:, 0] = z
    x.requires_grad_()
    w = torch.zeros((1, 8), dtype=dtype, device=gpu_device)
    w[0, 0] = 1
    h = gated_linear(x, w, torch.zeros_like(w), None, torch.ones(1, dtype=dtype, device=gpu_device), act)
    dx = torch.autograd.grad(h, x, torch.ones_like(h))[0][:, 0]
    zd = z.double()
    s, rest = torch.sigmoid(zd), torch.sigmoid(-zd)
    rel, flush = (2 * zd.abs() + 8) * R.U, 2.0 ** -126
    half, tiny = R.HALF_STEP[dtype], R.TINY[dtype]
    if act == "sigmoid":
        value, slope = s, s * rest
        e_value, e_slope = s * rel + flush, slope * 2 * rel + flush
    else:
        value, slope = zd * s, s * (1 + zd * rest)
        e_value = zd.abs() * (s * (rel + R.U) + flush)
        e_slope = slope.abs() * (rel + 2 * R.U) + s * zd.abs() * (s * rel + 4 * R.U) + s * 4 * R.U + flush * (1 + zd.abs())
    R.within(h[:, 0], value, half * value.abs() + 1.01 * e_value + tiny, act)
    R.within(dx, slope, half * slope.abs() + 1.01 * e_slope + tiny, act + "'s slope")
