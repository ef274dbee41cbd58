"""Gradients in fp16 whose factors -- da and du of the gated projection, ds and p of attention -- lie outside fp16's range
while the gradients themselves lie in it: as exact as where the factors are ordinary numbers.

Bounds: those of the operators' other tests, but for the smallest values.  There a factor is off by half a step of fp16 relative
to itself or, where that is subnormal, by 2^-24.  Here it is first multiplied by a power of two, so the second becomes a part of
the largest factor: 2^-38 of it where it was brought to 2^14 and more, and 2^-24 where the largest was inside 2^-6 .. 2^16
and left as it was."""
import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu

HALF, TINY = R.HALF_STEP[torch.float16], R.TINY[torch.float16]


def check_gated(dev, rows, dim, hidden, x_size, w_size, dh_size, up, bias, seed=0):
    from pixelsplat_amd.ops import gated_linear

    g = torch.Generator().manual_seed(seed)
    t = lambda *s, size: (torch.randn(s, generator=g) * size).half().to(dev)  # noqa: E731
    x, wg, wu = t(rows, dim, size=x_size), t(hidden, dim, size=w_size), t(hidden, dim, size=w_size)
    bg, bu = t(hidden, size=1.0), torch.full((hidden,), up, device=dev).half()
    dh = t(rows, hidden, size=dh_size)
    leaves = [x, wg, wu] + ([bg, bu] if bias else [])
    for p in leaves:
        p.requires_grad_()
    call = lambda: torch.autograd.grad(gated_linear(x, wg, wu, bg, bu, "silu"), leaves, dh)  # noqa: E731
    grads = call()
    assert all(torch.equal(p, q) for p, q in zip(grads, call()))
    xd, wgd, wud, bgd, bud, d = (p.detach().double() for p in (x, wg, wu, bg, bu, dh))
    _, want, mid = R.gated_linear(xd, wgd, wud, bgd, bud, "silu", d)
    peak = max(mid["da"].abs().max().item(), mid["du"].abs().max().item())
    floor = 2.0 ** -24 if 2.0 ** -5 < peak < 65000 else max(2.0 ** -38 * peak, 2.0 ** -24 if peak < 2.0 ** -5 and peak > 2.0 ** -7
                                                            or 65000 <= peak <= 66000 else 0)
    ea, eu = ((dim + 2) * R.U * (xd.abs() @ w.abs().T + b.abs()) for w, b in ((wgd, bgd), (wud, bud)))
    own = 16 * R.U
    value_err = 1.13 * ea + own * (mid["a"].abs() + 1)
    da_err = d.abs() * (1.13 * eu + mid["u"].abs() * (1.13 * ea + own)) + 8 * R.U * mid["da"].abs()
    du_err = d.abs() * value_err + 4 * R.U * mid["du"].abs()
    da_in, du_in = da_err + HALF * mid["da"].abs() + floor, du_err + HALF * mid["du"].abs() + floor
    acc = lambda n, m: (n + 2) * R.U * m  # noqa: E731
    errs = dict(
        x=da_in @ wgd.abs() + du_in @ wud.abs() + acc(2 * hidden, mid["da"].abs() @ wgd.abs() + mid["du"].abs() @ wud.abs()),
        w_gate=da_in.T @ xd.abs() + acc(rows, mid["da"].abs().T @ xd.abs()),
        w_up=du_in.T @ xd.abs() + acc(rows, mid["du"].abs().T @ xd.abs()),
        b_gate=da_err.sum(0) + acc(300, mid["da"].abs().sum(0)), b_up=du_err.sum(0) + acc(300, mid["du"].abs().sum(0)))
    for n, got in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), grads):
        assert want[n].abs().max() < 65000, "the case asks for more than fp16 holds"
        R.within(got, want[n], HALF * want[n].abs() + 1.01 * errs[n] + TINY, "d" + n)
    return peak


@pytest.mark.parametrize("rows,dim,hidden,x,w", [(40, 64, 16, 0.01, 0.02), (3, 40, 50, 0.01, 0.02), (700, 77, 101, 0.005, 0.005),
                                                 (6100, 264, 3500, 0.001, 0.001), (129, 512, 700, 0.002, 0.002)])
def test_gated_factors_beyond_the_largest(gpu_device, rows, dim, hidden, x, w):
    """dh u of some 10^5, which is infinite in fp16, times weights and inputs that bring it back."""
    assert check_gated(gpu_device, rows, dim, hidden, x, w, 1000.0, 100.0, False) > 1e5


@pytest.mark.parametrize("rows,dim,hidden,x,w", [(40, 64, 16, 8.0, 1.0), (3, 40, 50, 8.0, 1.0), (700, 77, 101, 4.0, 1.0),
                                                 (6100, 264, 3500, 1.0, 0.1), (129, 512, 700, 1.0, 1.0)])
def test_gated_factors_below_the_smallest(gpu_device, rows, dim, hidden, x, w):
    """dh of 2^-21, da and du of 2^-16 at most, of which fp16 keeps a few bits, in sums of many."""
    assert check_gated(gpu_device, rows, dim, hidden, x, w, 2.0 ** -21, 0.01 / x, True) < 2.0 ** -6


def test_gated_infinities_stay_in_their_row(gpu_device):
    """A gradient with an infinity leaves the other rows' dx as finite and as exact as without it."""
    from pixelsplat_amd.ops import gated_linear

    g = torch.Generator().manual_seed(3)
    for size in (2.0 ** -14, 1.0, 1000.0):
        x = (torch.randn((200, 64), generator=g) * 0.01).half().to(gpu_device).requires_grad_()
        w = (torch.randn((32, 64), generator=g) * 0.01).half().to(gpu_device)
        b = torch.full((32,), 100.0, device=gpu_device).half()
        dh = (torch.randn((200, 32), generator=g) * size).half().to(gpu_device)
        dx = torch.autograd.grad(gated_linear(x, w, w, b, b), x, dh)[0]
        bad = dh.clone()
        bad[7, 3], bad[150, 9] = float("inf"), float("nan")
        got = torch.autograd.grad(gated_linear(x, w, w, b, b), x, bad)[0]
        keep = torch.ones(200, dtype=torch.bool, device=gpu_device)
        keep[[7, 150]] = False
        assert torch.isfinite(dx).all() and torch.equal(got[keep], dx[keep]) and not torch.isfinite(got[~keep]).any()
