"""Group norm with an activation (pixelsplat_amd.ops.group_norm) against 64 bits.

Bounds, from the arithmetic.  A result of type T is off by half a step of T relative to its value, and by the fp32
roundings before it: xh = (x - mean) rstd carries at most 4 (mean and rstd rounded once, a subtraction, a product; the
sums are 64-bit), the affine map 2 more, and an activation of slope at most 1.13 and its own evaluation 10 more, each
2^-24 of the largest intermediate.  16-bit GELU adds 1.5e-7 of |z| (its erf).  The parameters' gradients are sums: at
most 300 sequential fp32 additions of a thread and a block, so 320 roundings of the sum of magnitudes."""
import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(dev, shape, dtype, param, seed=0, mean=0.7):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * 1.5 + mean + torch.randn(c, generator=g)).to(dtype).to(dev)
    w = (1 + 0.3 * torch.randn(c, generator=g)).to(param).to(dev)
    b = (0.3 * torch.randn(c, generator=g)).to(param).to(dev)
    dy = torch.randn(shape, generator=g).to(dtype).to(dev)
    return x, w, b, dy


def check(x, w, b, dy, groups, act, eps=1e-5, view=lambda t: t):
    from pixelsplat_amd.ops import group_norm

    dtype = x.dtype
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = group_norm(view(x), groups, w, b, eps, act)
    assert y.is_contiguous() and y.dtype == dtype
    with torch.no_grad():
        assert torch.equal(group_norm(view(x), groups, w, b, eps, act), y)
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(group_norm(view(x), groups, w, b, eps, act), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))          # bit for bit

    xd, wd, bd = (t if t is None else t.detach().double().requires_grad_() for t in (x, w, b))
    ref = R.group_norm(view(xd), groups, wd, bd, eps, act)
    want = torch.autograd.grad(ref, [t for t in (xd, wd, bd) if t is not None], dy.double())
    with torch.no_grad():
        pre = R.group_norm(view(xd), groups, None, None, eps, "none")
        wmax = 1.0 if w is None else wd.abs().max().item()
        bmax = 0.0 if b is None else bd.abs().max().item()
        n, c = pre.shape[0], pre.shape[-1]
        top = pre.abs().max().item() * wmax + bmax + 1
        # a mean far from zero: x - mean loses what the rounding of the mean is off by
        xg = view(xd).detach().reshape(n, -1, groups, c // groups)
        rstd = 1 / torch.sqrt(xg.var((1, 3), unbiased=False, keepdim=True) + eps)
        shift = (xg.mean((1, 3), keepdim=True).abs() * rstd).max().item() * wmax
        arith = R.U * (16 * top + shift) + (1.5e-7 * top if act == "gelu" and dtype != torch.float32 else 0)
        half = R.HALF_STEP[dtype]
        R.within(y, ref, half * ref.abs() + 2 * arith + R.TINY[dtype], "y")
        slope_err = 2 * arith if act != "relu" else 2 * arith          # |act''| <= 1
        dmax = dy.double().abs().max().item()
        if act == "relu":      # the slope jumps at 0: elements that near it are not compared
            near = ((pre * (1 if wd is None else wd) + (0 if bd is None else bd)).abs() < arith)
            assert near.double().mean() < 1e-3
        else:
            near = torch.zeros_like(pre, dtype=torch.bool)
        scale = rstd.max().item() * dmax * wmax * (2 + pre.abs().max().item())
        dx_bound = half * want[0].abs() + scale * (40 * R.U + slope_err) + R.TINY[dtype]
        keep = ~near if view(xd).shape == pre.shape else None
        got0 = view(grads[0]) if grads[0].shape != ref.shape else grads[0]
        want0 = view(want[0]) if want[0].shape != ref.shape else want[0]
        bound0 = view(dx_bound) if dx_bound.shape != ref.shape else dx_bound
        R.within(torch.where(keep, got0.double(), want0), want0, bound0, "dx")
        dz = dy.double().abs() * 1.13
        dims = tuple(range(dz.dim() - 1))
        sums = [(dz * pre.abs()).sum(dims), dz.sum(dims)]
        rest = [t for t, s in zip((x, w, b), (0, 1, 2)) if t is not None][1:]
        names = [nm for nm, t in (("dweight", w), ("dbias", b)) if t is not None]
        pick = [s for s, t in zip(sums, (w, b)) if t is not None]
        for nm, t, got, ref_g, mass in zip(names, rest, grads[1:], want[1:], pick):
            jump = (near * dz * (pre.abs() + 1)).sum(dims) if act == "relu" else 0
            R.within(got, ref_g, R.HALF_STEP[t.dtype] * ref_g.abs() + mass * (320 * R.U + slope_err) + jump
                     + R.TINY[t.dtype], nm)


# (shape, groups): the one-launch form, chunks, one row, one element, odd channels and groups, groups wider than a
# block's columns, one group, one channel a group, more columns than a block has
SHAPES = [((2, 16, 16, 128), 8), ((3, 40, 50, 128), 32), ((1, 1, 64), 4), ((4, 96), 12), ((1, 1), 1),
          ((2, 7, 9, 30), 5), ((3, 5, 77), 7), ((1, 33, 2056), 1), ((2, 19, 2056), 257), ((1, 3001, 24), 3),
          ((70, 9, 64), 2), ((1, 5, 8192), 8192), ((2, 130, 4200), 10)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_against_64_bits(gpu_device, shape, groups, dtype):
    act = ("none", "relu", "silu", "gelu", "sigmoid")[(len(shape) + groups + shape[-2]) % 5]
    check(*make(gpu_device, shape, dtype, dtype), groups, act)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 4), ((2, 61, 30), 3)], ids=str)
def test_activations_and_fp32_parameters(gpu_device, shape, groups, dtype, act):
    check(*make(gpu_device, shape, dtype, torch.float32, seed=3), groups, act)


@pytest.mark.parametrize("which", ["weight", "bias", "neither"])
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 4), ((2, 61, 30), 3)], ids=str)
def test_parameters_are_optional(gpu_device, shape, groups, which):
    x, w, b, dy = make(gpu_device, shape, torch.float32, torch.float32, seed=4)
    check(x, w if which == "weight" else None, b if which == "bias" else None, dy, groups, "silu")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("groups,c", [(4, 64), (3, 48), (2, 18)])
def test_strides(gpu_device, dtype, groups, c):
    """A slice of wider rows, every other row, a channels-first memory, and a misaligned start."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((3, 22, 2 * c + 8), generator=g).to(dtype).to(gpu_device)
    _, w, b, dy = make(gpu_device, (3, 22, c), dtype, dtype, seed=6)
    for view in (lambda t: t[..., 8:8 + c], lambda t: t[..., 1:1 + c]):
        check(wide.clone(), w.clone(), b.clone(), dy, groups, "gelu", view=view)
    check(wide.clone(), w.clone(), b.clone(), dy[:, ::2].contiguous(), groups, "gelu", view=lambda t: t[:, ::2, :c])
    first = torch.randn((3, c, 22), generator=g).to(dtype).to(gpu_device)
    check(first, w.clone(), b.clone(), dy, groups, "gelu", view=lambda t: t.transpose(1, 2))


def test_expanded_gradient_and_far_mean(gpu_device):
    from pixelsplat_amd.ops import group_norm

    x, w, b, _ = make(gpu_device, (2, 300, 64), torch.float32, torch.float32, seed=7, mean=3000.0)
    check(x, w, b, torch.randn((2, 300, 64), device=gpu_device), 4, "none")
    x = x.detach().requires_grad_()
    group_norm(x, 4, w, b).sum().backward()            # dy: one element, expanded
    ones = torch.ones((2, 300, 64), device=gpu_device)
    assert torch.equal(x.grad, torch.autograd.grad(group_norm(x, 4, w, b), x, ones)[0])


def test_constant_groups_and_nan(gpu_device):
    from pixelsplat_amd.ops import group_norm

    x = torch.full((2, 50, 32), 3.0, device=gpu_device, requires_grad=True)
    b = torch.randn(32, device=gpu_device)
    y = group_norm(x, 4, None, b, activation="none")
    assert torch.equal(y, b.expand_as(y))
    y.square().sum().backward()
    assert torch.isfinite(x.grad).all()
    for n in (50, 5000):                               # a NaN stays inside its sample and group
        x = torch.randn((2, n, 32), device=gpu_device)
        x[1, 7, 9] = float("nan")
        for act in ("none", "relu", "silu", "gelu", "sigmoid"):
            bad = group_norm(x, 4, activation=act).isnan()
            assert bad[1, :, 8:16].all() and bad.sum() == n * 8


def test_empty(gpu_device):
    from pixelsplat_amd.ops import group_norm

    for shape in ((0, 4, 8), (2, 0, 8)):
        x = torch.zeros(shape, device=gpu_device, requires_grad=True)
        w = torch.ones(8, device=gpu_device, requires_grad=True)
        y = group_norm(x, 2, w, None, activation="relu")
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and torch.equal(w.grad, torch.zeros_like(w))


def test_module_equals_library_group_norm(gpu_device):
    from pixelsplat_amd.ops import GroupNormAct

    net = GroupNormAct(4, 32, activation="gelu").to(gpu_device)
    with torch.no_grad():
        net.weight.normal_()
        net.bias.normal_()
    x = torch.randn((2, 32, 9, 11), device=gpu_device).to(memory_format=torch.channels_last)
    y = net(x)
    assert y.is_contiguous(memory_format=torch.channels_last)
    ref = torch.nn.functional.gelu(torch.nn.functional.group_norm(x.double(), 4, net.weight.double(), net.bias.double()))
    R.within(y, ref, 64 * R.U * ref.abs().max(), "module")
    assert set(net.state_dict()) == {"weight", "bias"}


def test_other_stream_and_graph(gpu_device):
    """On a side stream, and captured: every replay, with eager work between, equals the eager result."""
    from pixelsplat_amd.ops import group_norm

    for shape in ((2, 16, 16, 128), (2, 70, 50, 96)):
        x, w, b, dy = make(gpu_device, shape, torch.bfloat16, torch.float32, seed=8)
        for t in (x, w, b):
            t.requires_grad_()

        def step():
            y = group_norm(x, 8, w, b, activation="silu")
            return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(4):
            with torch.no_grad():
                x.copy_(torch.randn(shape, device=gpu_device))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, step())), i
