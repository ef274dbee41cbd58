"""The image-transformer operators with tensors that do not lie together: refused before anything is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_mixed_devices_are_refused(gpu_device):
    from pixelsplat_amd.ops import gated_linear, group_norm, relative_attention

    x, w, cpu = torch.zeros((3, 8), device=gpu_device), torch.zeros((5, 8), device=gpu_device), torch.zeros((5, 8))
    with pytest.raises(RuntimeError, match="w_up is on cpu"):
        gated_linear(x, w, cpu)
    with pytest.raises(RuntimeError, match="b_gate is on cpu"):
        gated_linear(x, w, w, cpu[:, 0])
    with pytest.raises(RuntimeError, match="bias is on cpu"):
        group_norm(x, 2, None, cpu[0])
    q = torch.zeros((1, 1, 4, 8), device=gpu_device)
    buckets = torch.zeros((1, 7), dtype=torch.int32, device=gpu_device)
    with pytest.raises(RuntimeError, match="buckets is on cpu"):
        relative_attention(q, q, q, x[:, :1], buckets.cpu())
    with pytest.raises(RuntimeError, match="key_mask is on cpu"):
        relative_attention(q, q, q, x[:, :1], buckets, torch.ones((1, 4), dtype=torch.bool))


def test_second_derivatives_are_refused(gpu_device):
    from pixelsplat_amd.ops import gated_linear, group_norm, relative_attention

    x = torch.randn((4, 8), device=gpu_device, requires_grad=True)
    q = torch.randn((1, 1, 4, 8), device=gpu_device, requires_grad=True)
    buckets = torch.zeros((1, 7), dtype=torch.int32, device=gpu_device)
    for y, leaf in ((group_norm(x, 2), x), (gated_linear(x, x, x), x), (relative_attention(q, q, q, x[:, :1], buckets), q)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_saved_tensors_notice_changes_in_place(gpu_device):
    from pixelsplat_amd.ops import gated_linear, group_norm

    for op in (lambda x: group_norm(x, 2), lambda x: gated_linear(x, x.detach().clone(), x.detach().clone())):
        leaf = torch.randn((4, 8), device=gpu_device, requires_grad=True)
        x = leaf * 1
        y = op(x)
        x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
