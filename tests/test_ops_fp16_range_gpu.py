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


def attention_case(dev, heads, grid, dim, queries, start, masked, q_size, k_size, v_size, do_size, grow=0, seed=0):
    """fp16 tensors of the given sizes; grow: v and do rise by that many powers of two along the tokens."""
    from pixelsplat_amd.ops import relative_bucket_count, relative_buckets

    g = torch.Generator().manual_seed(seed)
    n = grid[0] * grid[1]
    nq = queries or n
    t = lambda m, size: (torch.randn((2, heads, m, dim), generator=g) * size)  # noqa: E731
    rise = lambda m: torch.exp2(grow * (torch.arange(m) / m - 1))[:, None]  # noqa: E731
    q, k, v, do = t(nq, q_size), t(n, k_size), t(n, v_size) * rise(n), t(nq, do_size) * rise(nq)
    table = 0.3 * torch.randn((relative_bucket_count(grid, 8), heads), generator=g)
    mask = torch.rand((2, n), generator=g) < 0.7 if masked else None
    half = [x.half().to(dev) for x in (q, k, v)]
    return [*half, table.to(dev)], relative_buckets(grid, 8, device=dev), None if mask is None else mask.to(dev), start, \
        do.half().to(dev)


# heads, grid, dim, queries, first query, masked, sizes of q, k, v and do, growth
T5 = 2.0 ** -5
BEYOND = [(2, (2, 2), 64, None, 0, False, 0.1, 0.005, 100.0, 1000.0, 0),
          (1, (3, 40), 32, None, 0, True, 0.05, 0.005, 200.0, 1000.0, 0),
          (2, (1, 500), 128, 300, 100, False, 0.02, 0.01, 1500.0, 2000.0, 12)]
BELOW = [(2, (16, 16), 64, None, 0, False, T5, 32.0, 1.0, 2.0 ** -18, 0),
         (1, (40, 50), 32, None, 0, True, 32.0, T5, 1.0, 2.0 ** -14, 0),
         (1, (1, 6000), 64, 100, 3000, False, T5, 32.0, 1.0, 2.0 ** -10, 6),
         (2, (9, 30), 20, 33, 5, True, 32.0, T5, 1.0, 2.0 ** -16, 10),
         (1, (1, 40000), 16, 300, 20000, False, 1.0, 1.0, 1.0, 1.0, 0)]


@pytest.mark.parametrize("case", BEYOND + BELOW, ids=str)
def test_attention_factors_of_any_size(gpu_device, case):
    """ds beyond 65504 and where fp16 has few bits, also rising along what is summed; p of a hundred thousandth."""
    from pixelsplat_amd.ops import relative_attention
    from tests.test_ops_relative_attention_gpu import bounds

    t, buckets, mask, start, do = attention_case(gpu_device, *case)
    leaves = [x.requires_grad_() for x in t]
    call = lambda: torch.autograd.grad(  # noqa: E731
        relative_attention(*leaves, buckets, key_mask=mask, query_start=start), leaves, do)
    grads = call()
    assert all(torch.equal(x, y) for x, y in zip(grads, call()))
    scale = t[0].shape[3] ** -0.5
    _, want, _, e = bounds(t, buckets, mask, start, do, scale, torch.float16)
    qd, kd, vd, td = (x.detach().double() for x in t)
    ds = R.relative_attention(qd, kd, vd, td, buckets, mask, scale, start, do.double())[2]["ds"].abs()
    if case in BEYOND:
        assert ds.max() > 66000
    if mask is not None:
        kd = kd * mask[:, None, :, None]
    # what `bounds` allows for subnormal factors, 2^-24, becomes 2^-38 of the row's or column's largest (p: of 1)
    for i, (top, other) in enumerate(((ds.amax(3, keepdim=True), kd), (ds.amax(2, keepdim=True).transpose(2, 3), qd))):
        e[i] = e[i] + scale * (2.0 ** -38 * top - TINY) * other.abs().sum(2, keepdim=True)
    e[2] = e[2] + (2.0 ** -38 - TINY) * do.double().abs().sum(2, keepdim=True)
    for name, got, w, bound in zip(("dq", "dk", "dv", "dtable"), grads, want, e):
        assert name == "dtable" or w.abs().max() < 65000, "the case asks for more than fp16 holds"
        R.within(got, w, bound, name)


def test_attention_infinities_stay_in_their_row(gpu_device):
    """An infinite and a NaN gradient leave the other queries' dq as it was."""
    from pixelsplat_amd.ops import relative_attention

    for case in (BEYOND[1], BELOW[1]):
        t, buckets, mask, start, do = attention_case(gpu_device, *case)
        q = t[0].requires_grad_()
        call = lambda d: torch.autograd.grad(  # noqa: E731
            relative_attention(*t, buckets, key_mask=mask, query_start=start), q, d)[0]
        want = call(do)
        bad = do.clone()
        bad[0, 0, 5, 3], bad[1, 0, 70, 0] = float("inf"), float("nan")
        got = call(bad)
        keep = torch.ones(q.shape[:3], dtype=torch.bool, device=gpu_device)
        keep[0, 0, 5] = keep[1, 0, 70] = False
        assert torch.isfinite(want).all() and torch.equal(got[keep], want[keep])
        assert not torch.isfinite(got[0, 0, 5]).any() and not torch.isfinite(got[1, 0, 70]).any()


@pytest.mark.parametrize("queries", [1, 40, 1 << 16])
@pytest.mark.parametrize("below", [17.5, 20.0])
def test_attention_terms_far_below_the_largest(gpu_device, below, queries):
    """One key ahead of 2^18 others that are e^-17.5 (2^-25) or less each and together a good part of the result.  A term
    and what its rounding leaves are off by 2^-32 of the largest term at most where they are subnormal.  (Few queries split the
    keys, and then only one part holds that key; 2^16 do not.)"""
    from pixelsplat_amd.ops import relative_attention, relative_buckets
    from tests.test_ops_relative_attention_gpu import bounds

    n = 1 << 18
    q = torch.zeros((1, 1, queries, 16), dtype=torch.float16, device=gpu_device)
    k, v = torch.zeros((2, 1, 1, n, 16), dtype=torch.float16, device=gpu_device)
    q[..., 0] = 1
    k[..., 777, 0] = below
    v[:] = 1
    v[..., 777, :] = 0
    table = torch.zeros((8, 1), dtype=torch.float16, device=gpu_device)
    buckets = relative_buckets((1, n), 8, device=gpu_device)
    ref, _, e, _ = bounds([q[:, :, :1], k, v, table], buckets, None, 0, torch.zeros_like(q[:, :, :1]), 1.0, torch.float16)
    ref, e = ref.expand(q.shape), e.expand(q.shape)                  # every query is the same
    bound = e + (2.0 ** -31 - TINY) * v.double().abs().sum(2, keepdim=True)
    assert (bound < ref / 2).all()                       # a lost sum would be seen
    R.within(relative_attention(q, k, v, table, buckets, scale=1.0), ref, bound, "out")
    R.within(relative_attention(q.requires_grad_(), k, v, table, buckets, scale=1.0), ref, bound, "out in training")


def test_ranges_in_a_graph_and_on_another_stream(gpu_device):
    """A captured training step of both operators, replayed with gradients of other sizes: the range is chosen in each replay."""
    from pixelsplat_amd.ops import gated_linear, relative_attention

    t, buckets, mask, start, do = attention_case(gpu_device, 2, (6, 20), 32, None, 0, True, 0.1, 0.1, 1.0, 1.0)
    g = torch.Generator().manual_seed(4)
    x = (torch.randn((300, 64), generator=g) * 0.01).half().to(gpu_device)
    w = (torch.randn((96, 64), generator=g) * 0.01).half().to(gpu_device)
    b = torch.full((96,), 50.0, device=gpu_device).half()
    dh = torch.randn((300, 96), generator=g).half().to(gpu_device)
    leaves = [p.requires_grad_() for p in (*t, x, w)]

    def step():
        y, h = relative_attention(*leaves[:4], buckets, key_mask=mask), gated_linear(x, w, w, b, b)
        return [*torch.autograd.grad(y, leaves[:4], do), *torch.autograd.grad(h, leaves[4:], dh)]

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
    for i, size in enumerate((1.0, 2.0 ** -14, 800.0, 2.0 ** -10, 1.0, 800.0)):
        with torch.no_grad():
            do.copy_((torch.randn(do.shape, generator=g) * size).half())
            dh.copy_((torch.randn(dh.shape, generator=g) * size).half())
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(out, eager)), (i, size)
