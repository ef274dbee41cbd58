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
