"""Group norm over samples of very many rows (pixelsplat_amd.ops.group_norm)."""
import math

import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu

PART = 1 << 27


def test_the_longest_sample(gpu_device):
    """2^31 - 1 rows of one channel, whose last chunk ends beyond what 32 bits hold: every row is written and counted.

    Values are +1 and -1 in turn and 3 in the last 2^23 rows; dy is 1 in these and 0 elsewhere.  So mean, variance and the
    gradients' sums are known exactly.  Bounds: y and dx are rounded to fp16 (half a step), xh carries 4 roundings of
    fp32, dx 8 of terms of at most rstd (1 + 2 |xh|); d_beta and d_gamma as in the sums of shorter samples."""
    from pixelsplat_amd.ops import group_norm

    n, tail = (1 << 31) - 1, 1 << 23
    x = torch.ones((1, n, 1), dtype=torch.float16, device=gpu_device)
    x[:, 1::2] = -1
    x[:, -tail:] = 3
    plus = (n - tail + 1) // 2
    total, squares = plus - (n - tail - plus) + 3 * tail, n - tail + 9 * tail
    mean = total / n
    rstd = 1 / math.sqrt(squares / n - mean * mean + 1e-5)
    w = torch.ones(1, device=gpu_device, requires_grad=True)
    b = torch.zeros(1, device=gpu_device, requires_grad=True)
    x.requires_grad_()
    poison = torch.full_like(x, float("nan"))                  # what a row that is not written would hold
    del poison
    y = group_norm(x, 1, w, b)
    dy = torch.zeros_like(x)
    dy[:, -tail:] = 1
    poison = torch.full_like(x, float("nan"))
    del poison
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    top = (3 - mean) * rstd
    assert abs(db.item() - tail) <= 320 * R.U * tail
    assert abs(dw.item() - tail * top) <= 330 * R.U * tail * top
    m1, m2 = tail / n, tail * top / n
    half, tiny = R.HALF_STEP[torch.float16], R.TINY[torch.float16]
    for a in range(0, n, PART):
        part = slice(a, min(a + PART, n))
        xh = (x.detach()[0, part, 0].float() - mean) * rstd
        over = (y.detach()[0, part, 0].float() - xh).abs() - (half * xh.abs() + 8 * R.U * 4 + tiny)
        assert (over <= 0).all(), a                            # (a NaN is not)
        ref = rstd * (dy[0, part, 0].float() - m1 - xh * m2)
        over = (dx[0, part, 0].float() - ref).abs() - (half * ref.abs() + 400 * R.U * rstd * 8 + tiny)
        assert (over <= 0).all(), a


@pytest.mark.parametrize("c,groups,dtype", [(1, 1, torch.float32), (8, 2, torch.bfloat16)])
def test_sums_of_long_samples(gpu_device, c, groups, dtype):
    """The gradient's sums over 2^28 rows, of equal terms, whose roundings do not cancel: a thread adds 256 of them in fp32,
    and its sum, a block's and the result are rounded once each (260 roundings of 2^-24 of the sum at most)."""
    from pixelsplat_amd.ops import group_norm

    n = (1 << 28) // c
    x = torch.ones((1, n, c), dtype=dtype, device=gpu_device)
    x[:, ::2] = -1
    x.requires_grad_()
    w, b = torch.ones(c, device=gpu_device, requires_grad=True), torch.zeros(c, device=gpu_device, requires_grad=True)
    dy = torch.full((1, 1, 1), 0.7, dtype=dtype, device=gpu_device)
    dw, db = torch.autograd.grad(group_norm(x, groups, w, b), (w, b), dy.expand(1, n, c))
    want = n * dy.item()
    assert ((db.double() - want).abs() <= 260 * R.U * want).all(), (db.double() - want).abs().max().item() / want / R.U
    dw1 = torch.autograd.grad(group_norm(x, groups, w, b), w, x.detach())[0]      # xh = x rstd: terms of rstd
    want = n / math.sqrt(1 + 1e-5)
    assert ((dw1.double() - want).abs() <= 264 * R.U * want).all(), (dw1.double() - want).abs().max().item() / want / R.U


@pytest.mark.parametrize("shape,groups", [((65535, 2, 512), 512), ((32800, 1, 8192), 512)], ids=str)
def test_more_groups_than_a_launch_has_blocks(gpu_device, shape, groups):
    """2^24 (sample, group)s and more: one channel each (chunks of rows), and 32 bytes each (one launch)."""
    from tests.test_ops_group_norm_gpu import check, make

    check(*make(gpu_device, shape, torch.bfloat16, torch.float32, seed=9), groups, "none")
