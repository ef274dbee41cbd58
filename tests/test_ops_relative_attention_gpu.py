"""Attention with a relative position bias (pixelsplat_amd.ops.relative_attention) against 64 bits.

Bounds, from the arithmetic; u = 2^-24, half = half a step of the result's type, n keys, d the head's width.  A logit is
off by es = (d + 8) u scale |q|.|k| + 8 u |bias| (a product of d terms, the factor log2(e) on scale and bias, their
sum); a probability, relative to itself, by rel = 2 max(es) + (n + 24) u (its own logit and the others' in the sum,
exp2, the sum of up to n terms, its inverse).  16-bit types split p into its rounding and the rounded rest, off by
half^2, and by `tiny` where that is subnormal, before its product with v.  out: (rel + half^2 + (n + 2) u) sum p |v| +
tiny sum |v|, and half |out|.
dp: (d + 2) u |do|.|v|;  do.o: the same of |o| and the error of the unrounded o;  ds = p (dp - do.o): rel |ds| and p times
those two;  dq, dk, dv: sums of |error| |other| and of (n + 2) u |terms|, ds and p rounded by half and tiny first;
d_table: the sum of ds' errors over its pairs and (n + 64) u sum |ds|.
Underflow: fp32 instructions give 0 below 2^-126 = flush.  A row's sum has a term of at least 1, so p = exp2(..) / sum is
off by flush at most; ds = p (dp - do.o) by flush (|dp| + |do.o|) for p and flush for the product itself."""
import math

import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu

FLUSH = 2.0 ** -126
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(dev, batch, heads, grid, dim, dtype, queries=None, start=0, masked=False, per_axis=8, seed=0, table_type=None):
    from pixelsplat_amd.ops import relative_bucket_count, relative_buckets

    g = torch.Generator().manual_seed(seed)
    n = grid[0] * grid[1]
    nq = n if queries is None else queries
    t = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev)  # noqa: E731
    packed = t(batch, n, 3, heads, dim)
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
    q = q[:, :, start:start + nq]
    table = (0.7 * torch.randn((relative_bucket_count(grid, per_axis), heads), generator=g)).to(table_type or dtype).to(dev)
    buckets = relative_buckets(grid, per_axis, device=dev)
    mask = None
    if masked:
        mask = torch.rand((batch, n), generator=g) < 0.6
        mask[0, n // 2:] = False
        if batch > 1:
            mask[1] = False
        mask = mask.to(dev)
    return [q, k, v, table], buckets, mask, start, t(batch, nq, heads, dim).transpose(1, 2)


def bounds(tensors, buckets, mask, start, do, scale, dtype):
    q, k, v, table = (t.detach().double() for t in tensors)
    do = do.double()
    out, grads, mid = R.relative_attention(q, k, v, table, buckets, mask, scale, start, do)
    k, v, p = mid["k"], mid["v"], mid["p"]
    n, d, nq = k.shape[2], k.shape[3], q.shape[2]
    half = R.HALF_STEP[dtype]
    scale = abs(scale)                                         # below it scales magnitudes of errors
    own = 0.0 if dtype == torch.float32 else half
    tiny = 0.0 if dtype == torch.float32 else R.TINY[dtype]
    finite = torch.where(torch.isfinite(mid["bias"]), mid["bias"], torch.zeros_like(mid["bias"]))
    es = (d + 8) * R.U * scale * (q.abs() @ k.abs().transpose(-1, -2)) + 8 * R.U * finite.abs()
    if mask is not None:
        es = es.masked_fill(~mask[:, None, None], 0)
    rel = 2 * es.amax(-1, keepdim=True) + (n + 24) * R.U
    pv = p @ v.abs()
    o32 = (rel + (n + 2) * R.U + own ** 2) * pv + (tiny + FLUSH) * v.abs().sum(2, keepdim=True)
    e_out = o32 + half * out.abs() + R.TINY[dtype]
    e_dp = (d + 2) * R.U * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = ((d + 2) * R.U * do.abs() * out.abs() + do.abs() * o32).sum(-1, keepdim=True)
    ds = mid["ds"]
    e_ds = (rel + 8 * R.U) * ds.abs() + p * (e_dp + e_delta) + 8 * R.U * p * (mid["dp"].abs() + mid["delta"].abs()) + \
        FLUSH * (mid["dp"].abs() + mid["delta"].abs() + 1)
    e_in = e_ds + own * ds.abs() + tiny
    acc = lambda m: (m + 2) * R.U  # noqa: E731
    e_dq = scale * (e_in @ k.abs() + acc(n) * (ds.abs() @ k.abs()))
    e_dk = scale * (e_in.transpose(-1, -2) @ q.abs() + acc(nq) * (ds.abs().transpose(-1, -2) @ q.abs()))
    ep = (rel + own + acc(nq)) * p + tiny + FLUSH
    e_dv = ep.transpose(-1, -2) @ do.abs()
    grow = torch.zeros((table.shape[0] + 1, table.shape[1]), dtype=table.dtype, device=table.device)
    grow.index_add_(0, mid["flat"], (e_ds + (n + 64) * R.U * ds.abs()).sum(0).flatten(1).T)
    e = [e_dq, e_dk, e_dv, grow[:-1]]
    halves = [half, half, half, R.HALF_STEP[tensors[3].dtype]]
    return out, grads, e_out, [x + h * w.abs() + R.TINY[torch.float32] + (tiny if i < 3 else 0) + 4 * R.U * w.abs()
                               for i, (x, h, w) in enumerate(zip(e, halves, grads))]


def check(tensors, buckets, mask, start, do, scale=None):
    from pixelsplat_amd.ops import relative_attention

    dtype = do.dtype
    leaves = [t.detach().requires_grad_() for t in tensors]
    call = lambda ts: relative_attention(*ts, buckets, key_mask=mask, scale=scale, query_start=start)  # noqa: E731
    out = call(leaves)
    assert out.dtype == dtype and out.shape == leaves[0].shape
    with torch.no_grad():
        plain = call(leaves)
    grads = torch.autograd.grad(out, leaves, do)
    again = call(leaves)
    assert torch.equal(again, out) and all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(again, leaves, do), grads))
    s = leaves[0].shape[3] ** -0.5 if scale is None else scale
    ref, want, e_out, e_grads = bounds(tensors, buckets, mask, start, do, s, dtype)
    R.within(out, ref, e_out, "out")
    R.within(plain, ref, e_out, "out without gradients")
    for name, got, w, e in zip(("dq", "dk", "dv", "dtable"), grads, want, e_grads):
        R.within(got, w, e, name)
    return out, grads


# grid, dim, queries (None: all), first query
CASES = [((1, 1), 8, None, 0), ((1, 5), 16, None, 0), ((5, 1), 64, None, 0), ((3, 7), 40, None, 0), ((16, 16), 128, None, 0),
         ((9, 33), 64, None, 0), ((1, 200), 32, None, 0), ((2, 70), 72, None, 0), ((40, 3), 24, None, 0), ((1, 700), 64, None, 0),
         ((2, 512), 16, None, 0), ((8, 8), 20, None, 0), ((4, 5), 1, None, 0), ((7, 9), 33, None, 0),
         ((24, 24), 64, 1, 300), ((30, 40), 128, 1, 1199), ((16, 20), 64, 33, 100), ((1, 1500), 32, 7, 0), ((13, 64), 96, 70, 500)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("masked", [False, True], ids=["all", "masked"])
@pytest.mark.parametrize("grid,dim,queries,start", CASES)
def test_against_64_bits(gpu_device, grid, dim, queries, start, masked, dtype):
    check(*make(gpu_device, 2, 3, grid, dim, dtype, queries, start, masked))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_queries_and_few(gpu_device, dtype):
    """Enough blocks that the keys are not split, and one query of one head over a long sequence, which splits them far."""
    check(*make(gpu_device, 16, 8, (11, 17), 32, dtype, seed=1))
    check(*make(gpu_device, 1, 1, (1, 9000), 64, dtype, 1, 4500, seed=2))
    check(*make(gpu_device, 1, 1, (60, 80), 64, dtype, 2, 4700, masked=True, seed=3))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_last_round_of_few_blocks(gpu_device, dtype):
    """A few blocks more than there are CUs, which split what they stream: queries, keys or both in uneven parts."""
    check(*make(gpu_device, 3, 9, (33, 40), 32 if dtype == torch.float32 else 128, dtype, masked=True, seed=22))
    check(*make(gpu_device, 3, 9, (33, 40), 128, dtype, 1300, 11, seed=23))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("grid,queries,start", [((5, 64), None, 0), ((3, 96), 200, 33), ((6, 32), 64, 64), ((2, 128), 97, 128)])
def test_tiles_in_one_row_of_the_grid(gpu_device, grid, queries, start, dtype):
    """Grids as wide as tiles of keys and queries, wholly, partly and with the queries between two rows."""
    for masked in (False, True):
        check(*make(gpu_device, 2, 2, grid, 64, dtype, queries, start, masked, per_axis=40, seed=20))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_maximum_that_grows(gpu_device, dtype):
    """Logits that rise, jump and fall along the keys: by less than 8 powers of two a tile, by many, and back."""
    t, buckets, mask, start, do = make(gpu_device, 1, 2, (1, 640), 32, dtype, seed=21)
    n = torch.arange(640, device=gpu_device, dtype=torch.float32)
    for rise in (n / 40, -n / 40, 12 * (n // 64), 6 * torch.sin(n / 20)):
        q, k = t[0].clone(), t[1].clone()
        q[..., 0] = 1
        k[..., 0] = rise.to(dtype)
        check([q, k, t[2], t[3]], buckets, mask, start, do, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_offset_and_offsets_without_bias(gpu_device, dtype):
    """A map with a bucket for every offset, and one whose entries are partly outside the table."""
    t, _, mask, start, do = make(gpu_device, 2, 2, (6, 9), 32, dtype, seed=4)
    full = torch.arange(11 * 17, dtype=torch.int32).reshape(11, 17).to(gpu_device)
    g = torch.Generator().manual_seed(5)
    t[3] = torch.randn((11 * 17, 2), generator=g).to(dtype).to(gpu_device)
    check(t, full, mask, start, do)
    holes = full.clone()
    holes[::2, ::3] = -1
    holes[1, 1] = 11 * 17
    holes[2, 2] = 2 ** 31 - 1
    holes[3, 3] = -2 ** 31
    check(t, holes, mask, start, do)


def test_fp32_table_of_16_bit_tensors(gpu_device):
    for dtype in TYPES[1:]:
        _, grads = check(*make(gpu_device, 3, 2, (12, 12), 64, dtype, seed=6, table_type=torch.float32))
        assert grads[3].dtype == torch.float32


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scale(gpu_device, dtype):
    t, buckets, mask, start, do = make(gpu_device, 1, 2, (7, 10), 48, dtype, seed=7)
    check(t, buckets, mask, start, do, scale=0.03)
    check(t, buckets, mask, start, do, scale=0.0)
    check(t, buckets, mask, start, do, scale=-0.2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(gpu_device, dtype):
    """Head-major tensors, misaligned rows, expanded keys and an expanded gradient."""
    from pixelsplat_amd.ops import relative_attention

    t, buckets, mask, start, do = make(gpu_device, 2, 4, (5, 13), 32, dtype, masked=True, seed=8)
    want = relative_attention(*t, buckets, key_mask=mask)
    again = relative_attention(*(x.contiguous() for x in t), buckets, key_mask=mask)
    assert torch.equal(want, again)
    odd = [torch.cat([x[..., :1], x], -1)[..., 1:] for x in t[:3]]
    assert odd[0].data_ptr() % 16 and torch.equal(relative_attention(*odd, t[3], buckets, key_mask=mask), want)
    lying = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in t[:3]]
    assert torch.equal(relative_attention(*lying, t[3], buckets, key_mask=mask), want)
    assert torch.equal(relative_attention(*t, buckets, key_mask=mask.T.contiguous().T), want)
    shared = [t[0], t[1][:, :1].expand_as(t[1]), t[2][:, :1].expand_as(t[2]), t[3]]        # one head for all queries' heads
    check(shared, buckets, mask, start, do)
    leaf = [t[0].detach().requires_grad_(), t[1][:, :1].detach().requires_grad_(), t[2][:, :1].detach().requires_grad_(), t[3]]
    out = relative_attention(leaf[0], leaf[1].expand_as(t[1]), leaf[2].expand_as(t[2]), t[3], buckets, key_mask=mask)
    gk, gv = torch.autograd.grad(out, leaf[1:3], do)
    ref, wantg, _, e = bounds(shared, buckets, mask, start, do, 32 ** -0.5, dtype)
    for got, w, b in ((gk, wantg[1], e[1]), (gv, wantg[2], e[2])):       # the sum over heads, itself rounded
        total = w.sum(1, keepdim=True)
        R.within(got, total, b.sum(1, keepdim=True) + 4 * R.HALF_STEP[dtype] * w.abs().sum(1, keepdim=True), "shared head")
    q = t[0].detach().requires_grad_()
    y = relative_attention(q, *t[1:], buckets, key_mask=mask)
    a = torch.autograd.grad(y.sum(), q, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, q, torch.ones_like(y))[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_masked_keys_and_empty_rows_hold_anything(gpu_device, dtype):
    from pixelsplat_amd.ops import relative_attention

    for queries, start in ((None, 0), (1, 20)):
        t, buckets, mask, start, do = make(gpu_device, 3, 2, (6, 15), 64, dtype, queries, start, masked=True, seed=9)
        out, grads = check(t, buckets, mask, start, do)
        assert (out[1] == 0).all() and all((g[1] == 0).all() for g in grads[:3])
        assert all((g.transpose(1, 2)[~mask] == 0).all() for g in grads[1:3])
        bad = [x.clone() for x in t]
        for i, value in ((1, float("nan")), (2, float("inf"))):
            bad[i].transpose(1, 2)[~mask] = value
        do2 = do.clone()
        do2[1] = float("nan")                                  # upstream of rows without keys
        leaves = [x.detach().requires_grad_() for x in bad]
        again = relative_attention(*leaves, buckets, key_mask=mask, query_start=start)
        assert torch.equal(again, out)
        for got, want in zip(torch.autograd.grad(again, leaves, do2), grads):
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_biases_at_the_limits(gpu_device, dtype):
    """Buckets at minus infinity mask their offsets, also whole rows; a table at the type's lowest value is no bias at all."""
    from pixelsplat_amd.ops import relative_attention

    t, buckets, mask, start, do = make(gpu_device, 2, 2, (1, 90), 64, dtype, seed=10)
    lo = t[3].clone()
    lo[:] = torch.finfo(dtype).min
    if dtype == torch.float16:      # -65504 leaves its logits: q.k is lost beside it only in the wider types
        check([*t[:3], lo], buckets, mask, start, do)
    else:
        out, _ = check([*t[:3], lo], buckets, mask, start, do)      # every logit is that value: uniform
        mean = t[2].double().mean(2, keepdim=True)
        assert (out.double() - mean).abs().max() <= 0.01
    some = t[3].clone()
    some[0] = float("-inf")                                    # no token sees itself
    check([*t[:3], some], buckets, mask, start, do)
    none = torch.full_like(t[3], float("-inf"))
    out, grads = check([*t[:3], none], buckets, mask, start, do)
    assert (out == 0).all() and all((g == 0).all() for g in grads)
    far = t[3].clone()
    far[1:] = float("-inf")                                    # a token sees itself alone
    out = relative_attention(*t[:3], far, buckets)
    assert torch.equal(out, t[2])


def test_large_offsets(gpu_device):
    """Batch strides beyond 2^31 elements."""
    from pixelsplat_amd.ops import relative_attention

    t, buckets, _, start, do = make(gpu_device, 2, 2, (5, 8), 16, torch.bfloat16, seed=11)
    want = relative_attention(*t, buckets)
    leaves = [x.detach().requires_grad_() for x in t]
    grads = torch.autograd.grad(relative_attention(*leaves, buckets), leaves, do)
    room = torch.empty(((1 << 31) + 4096,), dtype=torch.bfloat16, device=gpu_device)
    far = [room[i * 1280:].as_strided((2, 2, 40, 16), (1 << 31, 16, 32, 1)) for i in range(3)]
    del room
    # the second element of each lies just behind 2^31 elements
    for x, y in zip(far, t):
        x.copy_(y)
    leaves = [x.detach().requires_grad_() for x in far] + [t[3].detach().requires_grad_()]
    out = relative_attention(*leaves, buckets)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, leaves, do), grads):
        assert torch.equal(a, b)


def test_only_what_is_asked_for(gpu_device):
    from pixelsplat_amd.ops import relative_attention

    t, buckets, mask, start, do = make(gpu_device, 2, 2, (7, 11), 32, torch.bfloat16, masked=True, seed=12)
    full = [x.detach().requires_grad_() for x in t]
    want = torch.autograd.grad(relative_attention(*full, buckets, key_mask=mask), full, do)
    for i in range(4):
        some = [x.detach().requires_grad_(j == i) for j, x in enumerate(t)]
        got = torch.autograd.grad(relative_attention(*some, buckets, key_mask=mask), some[i], do)[0]
        assert torch.equal(got, want[i])


def test_empty(gpu_device):
    from pixelsplat_amd.ops import relative_attention, relative_buckets

    table = torch.zeros((64, 2), device=gpu_device, requires_grad=True)
    k = torch.zeros((0, 2, 6, 8), device=gpu_device)
    y = relative_attention(k, k, k, table, relative_buckets((2, 3), 8, device=gpu_device))
    y.sum().backward()
    assert y.shape == k.shape and torch.equal(table.grad, torch.zeros_like(table))
    k = torch.zeros((2, 2, 6, 8), device=gpu_device)
    assert relative_attention(k[:, :, :0], k, k, table, relative_buckets((2, 3), 8, device=gpu_device)).shape == (2, 2, 0, 8)


def test_gradient_against_differences(gpu_device):
    from pixelsplat_amd.ops import relative_attention

    t, buckets, mask, start, do = make(gpu_device, 2, 2, (3, 5), 16, torch.float32, masked=True, seed=13)
    mask[1, 2:9] = True
    leaves = [x.detach().requires_grad_() for x in t]
    grads = torch.autograd.grad(relative_attention(*leaves, buckets, key_mask=mask), leaves, do)
    g = torch.Generator().manual_seed(14)
    for i, x in enumerate(t):
        d = torch.randn(x.shape, generator=g).to(gpu_device)
        e = 2.0 ** -7
        f = lambda s: (relative_attention(*[y + s * e * d if j == i else y for j, y in enumerate(t)], buckets,  # noqa: E731
                                          key_mask=mask).double() * do.double()).sum()
        diff, got = (f(1) - f(-1)) / (2 * e), (grads[i].double() * d.double()).sum()
        # the third-order term of a central difference (logits move by up to ~4 e a unit), and out's rounding over its step
        assert abs(diff - got) <= 200 * e * e * (1 + got.abs()) + 960 * 8 * R.U / e, i


def test_module(gpu_device):
    from pixelsplat_amd.ops import RelativePositionBias, relative_attention, relative_buckets

    net = RelativePositionBias(2, 8).to(gpu_device)
    with torch.no_grad():
        net.table.normal_()
    t, buckets, mask, _, _ = make(gpu_device, 2, 2, (4, 9), 32, torch.bfloat16, masked=True, seed=15)
    assert torch.equal(net(*t[:3], (4, 9), key_mask=mask), relative_attention(*t[:3], net.table, buckets, key_mask=mask))
    one = net(*(x[:, :, :9] for x in t[:3]), (1, 9))
    assert torch.equal(one, relative_attention(*(x[:, :, :9] for x in t[:3]), net.table[:8],
                                               relative_buckets((1, 9), 8, device=gpu_device)))


def test_other_stream_and_graph(gpu_device):
    from pixelsplat_amd.ops import relative_attention

    for dtype, grid, queries in ((torch.float32, (6, 20), None), (torch.bfloat16, (16, 20), None), (torch.float16, (30, 40), 1)):
        t, buckets, mask, start, do = make(gpu_device, 2, 2, grid, 64, dtype, queries, masked=True, seed=16)
        t = [x.detach().requires_grad_() for x in t]

        def step():
            y = relative_attention(*t, buckets, key_mask=mask)
            return [y.detach(), *torch.autograd.grad(y, t, do)]

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


def test_long_sequence(gpu_device):
    """More than 2^13 keys: against 64 bits at rows of its own, through the queries' block form."""
    from pixelsplat_amd.ops import relative_attention

    t, buckets, _, _, _ = make(gpu_device, 1, 1, (1, 20000), 32, torch.bfloat16, seed=17)
    out = relative_attention(*t, buckets)
    for start in (0, 9999, 19968):
        part = [t[0][:, :, start:start + 32], *t[1:]]
        do = torch.zeros_like(part[0])
        ref, _, e_out, _ = bounds(part, buckets, None, start, do, 32 ** -0.5, torch.bfloat16)
        R.within(out[:, :, start:start + 32], ref, e_out, f"rows {start}")
        R.within(relative_attention(*part, buckets, query_start=start), ref, e_out, f"block {start}")
    assert math.isfinite(out.float().abs().max().item())
