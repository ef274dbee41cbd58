"""The image-transformer operators as the encoder's modules use them: a block of image self-attention with a group norm on
its patches, a relative position bias and a gated feed-forward, in training, against the same modules in 64 bits of
plain torch; and a transformer over a padded batch, through the fused kernel and through a hook on its weights.

Tolerances.  fp32: a block is a chain of about 12 products of at most 256 terms; each adds up to 260 2^-24 of its sum of
magnitudes, which for these zero-mean sums is about sqrt(256) times the result, so 12 * 260 * 16 * 2^-24 = 3e-3 is the
worst case in the largest entry and 1e-4 of it (random signs: 1 / sqrt of the terms, twice) what is asked.  bf16: 14
tensors rounded one after the other, each by 2^-8 of the values and with random signs, sqrt(14) 2^-8 = 1.5e-2 in the norm
of the result, 3 times that in a gradient, which passes them twice."""
import copy

import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu


def plain_gated(self, x):
    return self.down(R.act(self.activation, self.gate(x)) * self.up(x))


def plain_attention(self, x, z=None, grid=None, key_mask=None):
    b, n, _ = x.shape
    q, k, v = (t.reshape(b, n, self.heads, -1).transpose(1, 2) for t in self.to_qkv(x).chunk(3, dim=-1))
    logits = q @ k.transpose(-1, -2) * self.scale + self.relative_bias.matrix(grid)
    if key_mask is not None:
        logits = logits.masked_fill(~key_mask[:, None, None], float("-inf"))
    p = torch.softmax(logits, -1).nan_to_num(0.0)
    return self.to_out((p @ v).transpose(1, 2).reshape(b, n, -1))


def plain_norm(self, x):
    return R.group_norm(x.movedim(1, -1), self.num_groups, self.weight, self.bias, self.eps, self.activation).movedim(-1, 1)


def in_64_bits(net):
    """A copy of `net` in double whose operators are plain torch."""
    from pixelsplat_amd.encoder import Attention, GatedFeedForward
    from pixelsplat_amd.ops import GroupNormAct

    twin = copy.deepcopy(net).double()
    for m in twin.modules():
        for kind, plain in ((GatedFeedForward, plain_gated), (Attention, plain_attention), (GroupNormAct, plain_norm)):
            if isinstance(m, kind):
                m.forward = plain.__get__(m)
    return twin


def far(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 1.5e-2)], ids=["fp32", "bf16"])
@pytest.mark.parametrize("hw", [(64, 64), (36, 52)], ids=str)
def test_image_self_attention_block(gpu_device, hw, dtype, tol):
    from pixelsplat_amd.encoder import ImageSelfAttentionCfg
    from pixelsplat_amd.encoder.epipolar_transformer import ImageSelfAttention

    torch.manual_seed(0)
    cfg = ImageSelfAttentionCfg(patch_size=4, num_octaves=10, num_layers=2, num_heads=4, d_token=128, d_dot=128, d_mlp=256,
                                relative_buckets=16, gated_mlp=True, norm_groups=8)
    net = ImageSelfAttention(cfg, 128, 128).to(gpu_device)
    with torch.no_grad():
        for p in net.parameters():
            if p.dim() == 1 or p.shape == (256, 4):
                p.add_(0.2 * torch.randn_like(p))
    net = net.to(dtype)
    x = torch.randn((2, 128, *hw), device=gpu_device).to(dtype).to(memory_format=torch.channels_last).requires_grad_()
    if dtype != torch.float32:       # the sin / cos positions stay what the module makes of fp32 coordinates
        net.positional_encoding[0].float()
        net.positional_encoding[0].register_forward_hook(lambda m, a, out: out.to(dtype))
    want_net = in_64_bits(net)
    if dtype != torch.float32:
        want_net.positional_encoding[0]._forward_hooks.clear()
    want_net.positional_encoding[0].float()
    want_net.positional_encoding[0].register_forward_hook(lambda m, a, out: out.to(dtype).double())
    dy = torch.randn_like(x)
    y = net(x)
    grads = torch.autograd.grad(y, [x, *net.parameters()], dy)
    xd = x.detach().double().requires_grad_()
    want = want_net(xd)
    want_grads = torch.autograd.grad(want, [xd, *want_net.parameters()], dy.double())
    assert far(y, want) <= tol
    names = ["x", *(n for n, _ in net.named_parameters())]
    for n, g, w in zip(names, grads, want_grads):
        assert g.dtype == dtype and far(g, w) <= 3 * tol, n


def test_transformer_on_a_padded_batch(gpu_device):
    """Rows of padding, one element of it padding alone: the fused path, the path that a hook on the weights takes, and
    64 bits; what the padding holds does not reach the tokens that are there."""
    from pixelsplat_amd.encoder import GatedFeedForward, Transformer

    torch.manual_seed(1)
    net = Transformer(64, 2, 2, 32, 96, feed_forward_layer=GatedFeedForward, relative_buckets=8).to(gpu_device)
    with torch.no_grad():
        for attn, _ in net.layers:
            attn.fn.relative_bias.table.normal_()
    lengths = torch.tensor([77, 30, 0, 1], device=gpu_device)
    mask = torch.arange(77, device=gpu_device)[None] < lengths[:, None]
    x = torch.randn((4, 77, 64), device=gpu_device)
    y = net(x, grid=(7, 11), key_mask=mask)
    want = in_64_bits(net)(x.double(), grid=(7, 11), key_mask=mask)
    assert far(y[mask], want[mask]) <= 1e-4
    other = torch.where(mask[..., None], x, torch.randn_like(x) * 50)
    assert torch.equal(net(other, grid=(7, 11), key_mask=mask)[mask], y[mask])
    seen = []
    for attn, _ in net.layers:
        attn.fn.attend.register_forward_hook(lambda m, a, out: seen.append(out))
    hooked = net(x, grid=(7, 11), key_mask=mask)
    assert len(seen) == 2 and seen[0].shape == (4, 2, 77, 77) and far(hooked[mask], want[mask]) <= 1e-4
    with pytest.raises(ValueError, match="grid"):
        net(x)
    with pytest.raises(ValueError, match="grid"):
        Transformer(64, 1, 2, 32, 96).to(gpu_device)(x, grid=(7, 11))


def test_refinement_norm(gpu_device):
    """The refinement convolutions' group norm + GELU in place of the GELU."""
    from pixelsplat_amd.encoder import EpipolarTransformer, EpipolarTransformerCfg, ImageSelfAttentionCfg
    from pixelsplat_amd.ops import GroupNormAct

    torch.manual_seed(2)
    sa = dict(patch_size=2, num_octaves=4, num_layers=1, num_heads=2, d_token=16, d_dot=8, d_mlp=32)
    cfg = EpipolarTransformerCfg(self_attention=ImageSelfAttentionCfg(**sa), num_octaves=10, num_layers=1, num_heads=2,
                                 num_samples=4, d_dot=8, d_mlp=32, downscale=2, refinement_groups=4)
    net = EpipolarTransformer(cfg, 16, num_context_views=2).to(gpu_device)
    assert isinstance(net.upscale_refinement[1], GroupNormAct)
    f = torch.randn((2, 16, 24, 20), device=gpu_device, requires_grad=True)
    y = net.upscale_refinement(f)
    twin = in_64_bits(net.upscale_refinement)
    fd = f.detach().double().requires_grad_()
    want = twin(fd)
    assert far(y, want) <= 1e-4
    dy = torch.randn_like(y)
    for g, w in zip(torch.autograd.grad(y, [f, *net.upscale_refinement.parameters()], dy),
                    torch.autograd.grad(want, [fd, *twin.parameters()], dy.double())):
        # a bias in front of a norm has almost no gradient: its size is measured by its neighbours'
        assert (g.double() - w).norm() <= 3e-4 * max(w.norm().item(), 1.0)


def test_whole_block_in_a_graph(gpu_device):
    """A captured training step of a block, replayed with other inputs: every replay equals the eager step."""
    from pixelsplat_amd.encoder import GatedFeedForward, Transformer

    torch.manual_seed(3)
    net = Transformer(64, 1, 2, 32, 96, feed_forward_layer=GatedFeedForward, relative_buckets=8).to(gpu_device)
    attn, ff = net.layers[0]
    q = [torch.randn((2, 2, 60, 32), device=gpu_device, requires_grad=True) for _ in range(3)]
    w = [ff.fn.gate.weight, ff.fn.up.weight, attn.fn.relative_bias.table]
    dy = torch.randn((2, 60, 96), device=gpu_device)

    def step():
        o = attn.fn.relative_bias(*q, (6, 10)).transpose(1, 2).reshape(2, 60, 64)
        return torch.autograd.grad(ff.fn.dropout(gated(o, ff.fn)), [*q, *w], dy)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    for i in range(4):
        with torch.no_grad():
            q[i % 3].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def gated(x, ff):
    from pixelsplat_amd.ops import gated_linear

    return gated_linear(x, ff.gate.weight, ff.up.weight, ff.gate.bias, ff.up.bias, ff.activation)
