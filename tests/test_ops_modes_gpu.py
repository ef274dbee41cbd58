"""The image-transformer operators under torch's modes and conventions: inference mode, autocast, changes in place."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_training_after_validation_in_inference_mode(gpu_device):
    """A module that has seen a grid in inference mode first trains on it, with the gradients of one that has not."""
    from pixelsplat_amd.encoder import GatedFeedForward, Transformer

    def grads(validate):
        torch.manual_seed(0)
        net = Transformer(32, 1, 2, 16, 48, feed_forward_layer=GatedFeedForward, relative_buckets=8).to(gpu_device)
        x = torch.randn((2, 20, 32), device=gpu_device)
        if validate:
            with torch.inference_mode():
                assert net(x, grid=(4, 5)).is_inference()
        net(x, grid=(4, 5)).square().sum().backward()
        return [p.grad for p in net.parameters()]

    for a, b in zip(grads(True), grads(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [32, 20, 1])
def test_results_changed_in_place(gpu_device, dim, dtype):
    """A result of attention is no view: a change in place is differentiated in 16-bit types, and noticed in fp32, whose
    backward pass reads the result itself."""
    from pixelsplat_amd.ops import relative_attention, relative_buckets

    g = torch.Generator().manual_seed(1)
    packed = torch.randn((2, 15, 3, 2, dim), generator=g).to(dtype).to(gpu_device)
    do = torch.randn((2, 15, 2, dim), generator=g).to(dtype).to(gpu_device).transpose(1, 2)
    table = torch.randn((64, 2), generator=g).to(dtype).to(gpu_device)
    buckets = relative_buckets((3, 5), 8, device=gpu_device)

    def call():
        leaf = packed.detach().requires_grad_()
        return leaf, relative_attention(*(leaf[:, :, i].transpose(1, 2) for i in range(3)), table, buckets)

    leaf, y = call()
    assert not y._is_view() and y.stride(3) == 1 and y.stride(1) < y.stride(2)
    want = torch.autograd.grad(y * 2, leaf, do)[0]
    leaf, z = call()
    z.mul_(2)
    assert torch.equal(z, y * 2)
    if dtype == torch.float32:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward(do)
    else:
        z.backward(do)
        assert torch.equal(leaf.grad, want)
    empty = packed[:0].detach().requires_grad_()
    q = empty[:, :, 0].transpose(1, 2)
    assert relative_attention(q, q, q, table, buckets).mul_(2).shape == (0, 2, 15, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_autocast(gpu_device, dtype):
    """Products take autocast's type, whatever their inputs and parameters are in; parameters' gradients come back in
    theirs.  A block of fp32 parameters trains behind a norm (fp32 there) and behind a projection (16 bits)."""
    from pixelsplat_amd.encoder import GatedFeedForward, Transformer
    from pixelsplat_amd.ops import gated_linear, group_norm, relative_attention, relative_buckets

    torch.manual_seed(2)
    x, w, b = (torch.randn(s, device=gpu_device, requires_grad=True) for s in ((6, 32), (2, 48, 32), (2, 48)))
    low = lambda t: t.detach().to(dtype).requires_grad_()  # noqa: E731
    xs, ws, bs = low(x), low(w), low(b)
    want = gated_linear(xs, *ws, *bs)
    dy = torch.randn_like(want)
    for given in (x, x.detach().to(dtype)):
        with torch.autocast("cuda", dtype):
            y = gated_linear(given, *w, *b)
        assert torch.equal(y, want)
        for got, ref in zip(torch.autograd.grad(y, (w, b), dy), torch.autograd.grad(want, (ws, bs), dy, retain_graph=True)):
            assert got.dtype == torch.float32 and torch.equal(got, ref.float())
    q, k, v = (torch.randn((2, 2, 15, 16), device=gpu_device) for _ in range(3))
    table = torch.randn((64, 2), device=gpu_device, requires_grad=True)
    buckets = relative_buckets((3, 5), 8, device=gpu_device)
    want = relative_attention(q.to(dtype), k.to(dtype), v.to(dtype), table, buckets)
    with torch.autocast("cuda", dtype):
        assert torch.equal(relative_attention(q, k.to(dtype), v, table, buckets), want)
        assert group_norm(x, 4).dtype == torch.float32
        with torch.autocast("cuda", enabled=False), pytest.raises(ValueError, match="w_gate is"):
            gated_linear(xs, *w)

    net = torch.nn.Sequential(torch.nn.Linear(32, 32), GatedFeedForward(32, 48)).to(gpu_device)
    block = Transformer(32, 1, 2, 16, 48, feed_forward_layer=GatedFeedForward, relative_buckets=8).to(gpu_device)
    for f in (lambda: net(torch.randn((2, 20, 32), device=gpu_device)),
              lambda: block(torch.randn((2, 20, 32), device=gpu_device), grid=(4, 5))):
        with torch.autocast("cuda", dtype):
            f().float().square().sum().backward()
    for p in [*net.parameters(), *block.parameters()]:
        assert p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0


def test_a_frozen_table_takes_no_room_for_its_gradient(gpu_device):
    """128 x 128 tokens: 2 x 128^4 / 8 bytes of sums for the table's gradient, none of them where it is not wanted."""
    from pixelsplat_amd.ops import relative_attention, relative_buckets

    buckets = relative_buckets((128, 128), 8, device=gpu_device)
    q = torch.randn((1, 1, 16384, 16), device=gpu_device).bfloat16().requires_grad_()
    table = torch.randn((64, 1), device=gpu_device)
    want = None
    for wanted in (True, False):
        y = relative_attention(q, q, q, table.requires_grad_(wanted), buckets)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = torch.autograd.grad(y, q, torch.ones_like(y))[0] if not wanted else \
            torch.autograd.grad(y, (q, table), torch.ones_like(y))[0]
        used = torch.cuda.max_memory_allocated() - before
        assert used > 2 * 16384 ** 2 // 8 if wanted else used < 32 << 20, (wanted, used)
        assert want is None or torch.equal(got, want)
        want = got
