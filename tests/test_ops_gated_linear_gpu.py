"""The gated projection (pixelsplat_amd.ops.gated_linear) against 64 bits.

Bounds, from the arithmetic; u = 2^-24, half = half a step of the result's type.  A product of k terms accumulated in
fp32 is off by at most (k + 2) u sum |terms| (the terms are exact for 16-bit operands, rounded once for fp32).  So the
projections a, u are off by Ea, Eu of that form; h by |u| |act'| Ea + |act| Eu + 16 u (|act| |u|) and half |h|.  The
gradients' factors da, du carry the same errors (|act'|, |act''| <= 1.13) and, in 16-bit types, half a step of their
own; a product over them is off by sum |their errors| |other| + (k + 2) u sum |terms|, and half of the result.  16-bit
GELU adds 1.5e-7 |a|."""
import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(dev, rows, dim, hidden, dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(dtype).to(dev)  # noqa: E731
    x, wg, wu = t(rows, dim), t(hidden, dim, scale=dim ** -0.5), t(hidden, dim, scale=dim ** -0.5)
    b = (t(hidden, scale=0.2), t(hidden, scale=0.2)) if bias else (None, None)
    return [x, wg, wu, *b], t(rows, hidden)


def check(tensors, dh, act, call=None):
    from pixelsplat_amd.ops import gated_linear

    call = call or (lambda *t: gated_linear(*t, activation=act))
    dtype = dh.dtype
    names = [n for n, t in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), tensors) if t is not None]
    leaves = [t.requires_grad_() for t in tensors if t is not None]
    h = call(*tensors)
    assert h.dtype == dtype and h.is_contiguous()
    with torch.no_grad():
        assert torch.equal(call(*tensors), h)
    grads = torch.autograd.grad(h, leaves, dh)
    again = torch.autograd.grad(call(*tensors), leaves, dh)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))

    x, wg, wu, bg, bu = (t if t is None else t.detach().double() for t in tensors)
    d = dh.double()
    ref, want, mid = R.gated_linear(x, wg, wu, bg, bu, act, d)
    half, k = R.HALF_STEP[dtype], x.shape[1]
    mass = lambda w, b: (x.abs() @ w.abs().T) + (0 if b is None else b.abs())  # noqa: E731
    ea, eu = (k + 2) * R.U * mass(wg, bg), (k + 2) * R.U * mass(wu, bu)
    own = 16 * R.U + (1.5e-7 if act == "gelu" and dtype != torch.float32 else 0)
    value_err = 1.13 * ea + own * (mid["a"].abs() + 1)
    h_err = mid["u"].abs() * value_err + mid["value"].abs() * eu + 4 * R.U * ref.abs()
    R.within(h, ref, half * ref.abs() + 2 * h_err + R.TINY[dtype], "h")
    # relu's slope jumps at 0: where a may be either side of it, da is either 0 or dh u
    jump = d.abs() * mid["u"].abs() * (mid["a"].abs() <= ea) if act == "relu" else 0
    round_own = half if dtype != torch.float32 else 0
    da_err = d.abs() * (1.13 * eu + mid["u"].abs() * (1.13 * ea + own)) + 8 * R.U * mid["da"].abs() + jump
    du_err = d.abs() * value_err + 4 * R.U * mid["du"].abs()
    da_in, du_in = da_err + round_own * mid["da"].abs() + R.TINY[dtype], du_err + round_own * mid["du"].abs() + R.TINY[dtype]
    rows, hidden = d.shape
    acc = lambda n, m: (n + 2) * R.U * m  # noqa: E731
    errs = dict(
        x=da_in @ wg.abs() + du_in @ wu.abs() + acc(2 * hidden, mid["da"].abs() @ wg.abs() + mid["du"].abs() @ wu.abs()),
        w_gate=da_in.T @ x.abs() + acc(rows, mid["da"].abs().T @ x.abs()),
        w_up=du_in.T @ x.abs() + acc(rows, mid["du"].abs().T @ x.abs()),
        b_gate=da_err.sum(0) + acc(300, mid["da"].abs().sum(0)),
        b_up=du_err.sum(0) + acc(300, mid["du"].abs().sum(0)))
    for n, got in zip(names, grads):
        R.within(got, want[n].reshape(got.shape), half * want[n].abs().reshape(got.shape)
                 + 1.01 * errs[n].reshape(got.shape) + R.TINY[dtype], "d" + n)


# rows, dim, hidden: one and a few rows, the tile's edges, odd everything, split contractions, the large tile
SIZES = [(1, 64, 96), (1, 1, 1), (3, 40, 130), (8, 128, 64), (9, 72, 65), (127, 128, 63), (129, 136, 129), (64, 33, 50),
         (700, 77, 101), (2000, 24, 40), (33, 512, 700), (5, 1000, 3)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,dim,hidden", SIZES)
def test_against_64_bits(gpu_device, rows, dim, hidden, dtype):
    act = ("silu", "gelu", "relu", "sigmoid", "none")[(rows + dim + hidden) % 5]
    check(*make(gpu_device, rows, dim, hidden, dtype, bias=hidden % 2 == 0), act)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid", "none"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_activations(gpu_device, dtype, act):
    check(*make(gpu_device, 200, 64, 80, dtype, seed=1), act)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_large_tiles(gpu_device, dtype):
    """Enough tiles for the 256 x 256 form in the forward and in both gradients' products."""
    check(*make(gpu_device, 6100, 264, 3500, dtype, seed=2), "silu")
    check(*make(gpu_device, 300, 5000, 6200, dtype, seed=3, bias=False), "gelu")


def test_many_rows(gpu_device):
    """More parts of 64 rows than a grid's second axis holds."""
    check(*make(gpu_device, (1 << 22) + 3, 8, 8, torch.float32, seed=12), "silu")


@pytest.mark.parametrize("which", ["gate", "up"])
def test_one_bias(gpu_device, which):
    t, dh = make(gpu_device, 70, 64, 48, torch.bfloat16, seed=4)
    t[4 if which == "gate" else 3] = None
    check(t, dh, "silu")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_shapes(gpu_device, dtype):
    from pixelsplat_amd.ops import gated_linear

    g = torch.Generator().manual_seed(5)
    wide = torch.randn((6, 7, 160), generator=g).to(dtype).to(gpu_device)
    packed = (torch.randn((2 * 50, 64), generator=g) / 8).to(dtype).to(gpu_device)
    b = torch.randn((100,), generator=g).to(dtype).to(gpu_device)
    for view in (lambda t: t[..., 32:96], lambda t: t[..., 3:67], lambda t: t.transpose(0, 1)[..., :64]):
        x = view(wide)
        y = gated_linear(x, packed[:50], packed[50:], b[:50], b[50:], "silu")
        want = gated_linear(x.contiguous(), packed[:50].clone(), packed[50:].clone(), b[:50].clone(), b[50:].clone(), "silu")
        assert y.shape == (*x.shape[:-1], 50) and torch.equal(y, want)
    x = wide[..., :64].detach().requires_grad_()
    w = packed.detach().requires_grad_()
    y = gated_linear(x, w[:50], w[50:], activation="gelu")
    gx, gw = torch.autograd.grad(y.sum(), (x, w))           # an expanded dh
    x2 = x.detach().reshape(-1, 64).double()
    _, want, _ = R.gated_linear(x2, packed[:50].double(), packed[50:].double(), None, None, "gelu",
                                torch.ones((42, 50), device=gpu_device).double())
    tol = 40 * R.HALF_STEP[dtype] if dtype != torch.float32 else 2e-5     # of the largest entry: sums of 42 .. 100 terms
    for got, ref in ((gx.reshape(-1, 64), want["x"]), (gw, torch.cat([want["w_gate"], want["w_up"]]))):
        R.within(got, ref, tol * ref.abs().max(), "strided gradient")
    # weights across: a transposed view is copied
    wt = (torch.randn((64, 50), generator=g) / 8).to(dtype).to(gpu_device)
    assert torch.equal(gated_linear(wide[..., :64], wt.T, packed[:50]), gated_linear(wide[..., :64], wt.T.contiguous(), packed[:50]))


def test_only_what_is_asked_for(gpu_device):
    from pixelsplat_amd.ops import gated_linear

    t, dh = make(gpu_device, 50, 64, 48, torch.bfloat16, seed=6)
    full = [p.clone().requires_grad_() for p in t]
    gated_linear(*full).backward(dh)
    for i in range(5):
        some = [p.clone().requires_grad_(j == i) for j, p in enumerate(t)]
        gated_linear(*some).backward(dh)
        assert torch.equal(some[i].grad, full[i].grad)


def test_nan_and_infinity_stay_in_their_row(gpu_device):
    """Rows that hold a NaN or an infinity leave every other row as it was, also in the same tile and behind the last row."""
    from pixelsplat_amd.ops import gated_linear

    for rows in (5, 140):
        for dtype in TYPES:
            t, _ = make(gpu_device, rows, 40, 70, dtype, seed=7)
            want = gated_linear(*t)
            x = t[0].clone()
            x[2, 39], x[rows - 1, 0] = float("nan"), float("inf")
            got = gated_linear(x, *t[1:])
            keep = torch.ones(rows, dtype=torch.bool)
            keep[[2, rows - 1]] = False
            assert torch.equal(got[keep], want[keep]) and got[2].isnan().all()


def test_empty(gpu_device):
    from pixelsplat_amd.ops import gated_linear

    w = torch.randn((6, 8), device=gpu_device, requires_grad=True)
    x = torch.zeros((0, 8), device=gpu_device, requires_grad=True)
    y = gated_linear(x, w, w)
    assert y.shape == (0, 6)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == (0, 8)
    assert gated_linear(torch.zeros((3, 8), device=gpu_device), w.detach()[:0], w.detach()[:0]).shape == (3, 0)


def test_gradient_against_differences(gpu_device):
    from pixelsplat_amd.ops import gated_linear

    t, dh = make(gpu_device, 12, 16, 20, torch.float32, seed=8)
    t = [p.requires_grad_() for p in t]
    grads = torch.autograd.grad(gated_linear(*t, activation="gelu"), t, dh)
    g = torch.Generator().manual_seed(9)
    for i, p in enumerate(t):
        v = torch.randn(p.shape, generator=g).to(gpu_device)
        e = 2.0 ** -7
        f = lambda s: (gated_linear(*[q.detach() + s * e * v if j == i else q.detach() for j, q in enumerate(t)],  # noqa: E731
                                    activation="gelu").double() * dh.double()).sum()
        # the third-order term of a central difference, and h's rounding over its step
        diff = (f(1) - f(-1)) / (2 * e)
        got = (grads[i].double() * v.double()).sum()
        assert abs(diff - got) <= 60 * e * e * (1 + got.abs()) + 240 * 8 * R.U / e, i


def test_other_stream_and_graph(gpu_device):
    from pixelsplat_amd.ops import gated_linear

    for dtype, rows in ((torch.float32, 300), (torch.bfloat16, 300), (torch.bfloat16, 2)):
        t, dh = make(gpu_device, rows, 64, 96, dtype, seed=10)
        t = [p.requires_grad_() for p in t]

        def step():
            h = gated_linear(*t)
            return [h.detach(), *torch.autograd.grad(h, t, dh)]

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
                t[0].copy_(torch.randn(t[0].shape, device=gpu_device))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, step())), i
