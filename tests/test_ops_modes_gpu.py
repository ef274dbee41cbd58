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
