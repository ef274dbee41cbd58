"""CPU checks of the image-transformer operators: the library builds and exports what its header declares, and every
refusal -- of the Python layer and of the C ABI -- is an error and no crash.  Nothing is launched."""
import ctypes as C
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from pixelsplat_amd.ops import build
    build.build()
    from pixelsplat_amd.ops import _lib
    return _lib.load()


def test_header_symbols_and_build_stamp(lib):
    from pixelsplat_amd.ops import _lib, build
    hdr = open(os.path.join(ROOT, "pixelsplat_amd", "ops", "include", "pixelsplat_ops.h")).read()
    hdr = re.sub(r"/\*.*?\*/", "", hdr, flags=re.S)
    names = set(re.findall(r"\b(ps_[a-z_0-9]+)\s*\(", hdr))
    assert names == set(_lib.SIGNATURES) and all(hasattr(lib, n) for n in names)
    assert build.unit_hashes() in lib.ps_ops_build_info().decode()


def test_missing_library_fails_loudly(monkeypatch, tmp_path):
    from pixelsplat_amd._lib import HipExtensionMissing
    from pixelsplat_amd.ops import _lib, group_norm
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(HipExtensionMissing):
        _lib.load()
    with pytest.raises(HipExtensionMissing):
        group_norm(torch.zeros(2, 3, 8), 2)


def test_group_norm_refusals(lib):
    from pixelsplat_amd.ops import GroupNormAct, group_norm
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm(x, 2)
    with pytest.raises(TypeError, match="Double"):
        group_norm(x.double(), 2)
    with pytest.raises(ValueError, match="activation"):
        GroupNormAct(2, 8, activation="tanh")


@pytest.mark.parametrize("kwargs,match", [
    (dict(num_groups=3), "do not divide"), (dict(num_groups=0), "do not divide"),
    (dict(num_groups=2, eps=-1.0), "eps"), (dict(num_groups=2, eps=float("nan")), "eps"),
    (dict(num_groups=2, activation="tanh"), "activation"),
    (dict(num_groups=2, weight=torch.ones(7)), "weight is"), (dict(num_groups=2, bias=torch.ones(8).half()), "bias is"),
    (dict(num_groups=2, bias=torch.ones(8).double()), "bias is")])
def test_group_norm_argument_refusals(lib, kwargs, match):
    from pixelsplat_amd.ops import group_norm
    with pytest.raises(ValueError, match=match):
        group_norm(torch.zeros(2, 3, 8), **kwargs)
    with pytest.raises(ValueError, match="different types"):
        group_norm(torch.zeros(2, 3, 8).half(), 2, torch.ones(8), torch.ones(8).half())
    with pytest.raises(ValueError, match="n, ..., channels"):
        group_norm(torch.zeros(8), 2)


def test_group_norm_c_abi_refusals(lib):
    from pixelsplat_amd.ops import _lib
    good = dict(samples=2, rows=6, channels=8, groups=2, dtype=0, activation=0, param_f32=1, eps=1e-5,
                x_sample_stride=48, x_row_stride=8, dy_sample_stride=48, dy_row_stride=8)
    p = 4096          # an address that is never followed
    ok = _lib.PsGroupNormDesc(**good)
    size = lib.ps_group_norm_workspace_bytes(C.byref(ok), 0)
    assert size > 0 and lib.ps_group_norm_workspace_bytes(C.byref(ok), 1) > 0

    def forward(d, x=p, y=p, ws=p, n=1 << 30):
        return lib.ps_group_norm_forward(C.byref(d) if d else None, x, None, None, y, p, p, ws, n, None)

    def backward(d, dy=p, dx=p, n=1 << 30):
        return lib.ps_group_norm_backward(C.byref(d) if d else None, p, dy, None, None, p, p, dx, None, None, p, n, None)

    assert forward(None) == backward(None) == -1
    assert forward(ok, x=None) == forward(ok, y=None) == forward(ok, ws=None) == forward(ok, y=p + 2) == -1
    assert backward(ok, dy=None) == backward(ok, dx=p + 8) == -1
    assert forward(ok, n=0) == backward(ok, n=0) == -2
    for field, value, status in [("samples", 0, -1), ("rows", 0, -1), ("rows", -4, -1), ("channels", 9, -1),
                                 ("groups", 0, -1), ("eps", -1.0, -1), ("x_row_stride", 7, -1), ("dtype", 3, -4),
                                 ("dtype", -1, -4), ("activation", 5, -4), ("samples", 70000, -4),
                                 ("rows", 1 << 28, -4)]:
        bad = _lib.PsGroupNormDesc(**{**good, field: value})
        assert forward(bad) == status and backward(bad) == status, field
        assert lib.ps_group_norm_workspace_bytes(C.byref(bad), 1) == 0


def test_gated_linear_refusals(lib):
    from pixelsplat_amd.ops import gated_linear
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_linear(x, w, w)
    with pytest.raises(TypeError, match="Int"):
        gated_linear(x.int(), w, w)
    fake = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)  # noqa: E731
    for args in [(fake(3, 8), fake(5, 7), fake(5, 7)), (fake(3, 8), fake(5, 8), fake(6, 8)), (fake(3, 8), fake(8), fake(8))]:
        with pytest.raises(ValueError, match="two weights"):
            gated_linear(*args)
    with pytest.raises(ValueError, match="w_up is"):
        gated_linear(fake(3, 8), fake(5, 8), fake(5, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="b_gate is"):
        gated_linear(fake(3, 8), fake(5, 8), fake(5, 8), fake(4))
    with pytest.raises(ValueError, match="activation"):
        gated_linear(fake(3, 8), fake(5, 8), fake(5, 8), activation="tanh")
    with pytest.raises(ValueError, match="dim is 0"):
        gated_linear(fake(3, 0), fake(5, 0), fake(5, 0))


def test_gated_linear_c_abi_refusals(lib):
    from pixelsplat_amd.ops import _lib
    good = dict(rows=6, dim=16, hidden=5, dtype=1, activation=2, reserved=0, x_row_stride=16, w_row_stride=16,
                dh_row_stride=5)
    p = 4096          # an address that is never followed
    ok = _lib.PsGatedLinearDesc(**good)
    assert lib.ps_gated_linear_backward_workspace_bytes(C.byref(ok)) > 0

    def forward(d, x=p, wu=p, h=p, gate=None, up=None):
        return lib.ps_gated_linear_forward(C.byref(d) if d else None, x, p, wu, None, None, h, gate, up, None)

    def backward(d, dh=p, gate=p, ws=p, n=1 << 40):
        return lib.ps_gated_linear_backward(C.byref(d) if d else None, p, p, p, None, None, gate, gate, dh, None, None,
                                            None, None, None, ws, n, None)

    assert forward(None) == backward(None) == forward(ok, x=None) == forward(ok, x=p + 2) == forward(ok, wu=p + 8) == -1
    assert forward(ok, h=None) == forward(ok, gate=p) == backward(ok, dh=None) == backward(ok, ws=p + 4) == -1
    assert backward(_lib.PsGatedLinearDesc(**{**good, "dtype": 0}), gate=None) == -1
    assert backward(ok, n=100) == -2
    for field, value, status in [("rows", 0, -1), ("dim", 0, -1), ("hidden", -1, -1), ("dim", 12, -1),
                                 ("x_row_stride", 8, -1), ("x_row_stride", 20, -1), ("w_row_stride", 17, -1),
                                 ("dtype", 3, -4), ("activation", 5, -4), ("rows", 1 << 30, -4)]:
        bad = _lib.PsGatedLinearDesc(**{**good, field: value})
        assert forward(bad) == status and backward(bad) == status, field
        assert lib.ps_gated_linear_backward_workspace_bytes(C.byref(bad)) == 0
    assert backward(_lib.PsGatedLinearDesc(**{**good, "dh_row_stride": 4})) == -1


def _attention_args(**changes):
    fake = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)  # noqa: E731
    a = dict(q=fake(2, 3, 6, 8), k=fake(2, 3, 6, 8), v=fake(2, 3, 6, 8), table=fake(5, 3),
             buckets=fake(3, 5, dtype=torch.int32))
    return {**a, **{n: fake(*c) if isinstance(c, tuple) else c for n, c in changes.items()}}


@pytest.mark.parametrize("changes,match", [
    (dict(k=(2, 3, 7, 8)), "q .batch"), (dict(q=(2, 3, 6)), "q .batch"), (dict(q=(2, 4, 6, 8)), "q .batch"),
    (dict(q=(2, 3, 6, 16)), "q .batch"), (dict(k=(2, 3, 7, 8), v=(2, 3, 7, 8)), "7 keys on a grid of 2 x 3"),
    (dict(q=(2, 3, 7, 8)), "queries 0 .. 6 of 6"), (dict(query_start=1), "queries 1 .. 6"), (dict(query_start=-1), "queries -1"),
    (dict(table=(5, 2)), "table is"), (dict(table=(0, 3)), "table is"), (dict(table=(3,)), "table is"),
    (dict(buckets=(3, 5)), "int32"), (dict(key_mask=(2, 6)), "bool")])
def test_relative_attention_refusals(lib, changes, match):
    from pixelsplat_amd.ops import relative_attention
    with pytest.raises(ValueError, match=match):
        relative_attention(**_attention_args(**changes))


def test_relative_attention_more_refusals(lib):
    from pixelsplat_amd.ops import RelativePositionBias, relative_attention, relative_buckets
    fake = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype)  # noqa: E731
    with pytest.raises(ValueError, match="buckets is"):
        relative_attention(**_attention_args(buckets=fake(4, 5, dtype=torch.int32)))
    with pytest.raises(ValueError, match="k and v are"):
        relative_attention(**_attention_args(v=fake(2, 3, 6, 8, dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="dim 136"):
        relative_attention(**_attention_args(q=(2, 3, 6, 136), k=(2, 3, 6, 136), v=(2, 3, 6, 136)))
    wide = dict(q=fake(1, 1, 1, 1), k=fake(1, 1, 1026, 1), v=fake(1, 1, 1026, 1), table=fake(5, 1),
                buckets=fake(3, 1025, dtype=torch.int32))
    with pytest.raises(ValueError, match="512 columns"):
        relative_attention(**wide)
    x = torch.zeros(1, 1, 1, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        relative_attention(x, x, x, torch.zeros(1, 1), torch.zeros(1, 1, dtype=torch.int32))
    for bad in (0, 6, -4):
        with pytest.raises(ValueError, match="multiple of 4"):
            RelativePositionBias(2, bad)
    with pytest.raises(ValueError, match="max_distance"):
        relative_buckets((4, 4), 32, 8)
    with pytest.raises(ValueError, match="at least one row"):
        relative_buckets((0, 4))


def test_relative_buckets():
    from pixelsplat_amd.ops import RelativePositionBias, relative_bucket_count, relative_buckets
    b = relative_buckets((1, 300), 32, 128)[0]
    at = lambda d: int(b[d + 299])  # noqa: E731
    assert [at(-d) for d in range(8)] == list(range(8)) and [at(d) for d in range(1, 8)] == list(range(17, 24))
    assert at(-8) == 8 and at(-15) == 9 and at(-16) == 10 and at(-299) == at(-128) == 15 and at(128) == at(299) == 31
    # far distances 8 16^(j / 8): 8, 11.3, 16, 22.6, 32, 45.3, 64, 90.5
    assert [at(-d) for d in (11, 12, 22, 23, 31, 32, 45, 46, 63, 64, 90, 91)] == [8, 9, 10, 11, 11, 12, 12, 13, 13, 14, 14, 15]
    two = relative_buckets((3, 4), 8)
    assert two.shape == (5, 7) and two.dtype == torch.int32
    assert int(two[2, 3]) == 0 and int(two[2, 4]) == 5 and int(two[3, 3]) == 40 and int(two[0, 0]) == 2 * 8 + 2
    assert int(two.max()) < relative_bucket_count((3, 4), 8) == 64
    assert relative_bucket_count((1, 9)) == relative_bucket_count((9, 1)) == 32 and relative_bucket_count((1, 1)) == 1
    net = RelativePositionBias(2, 8)
    assert torch.equal(net.buckets((3, 4), "cpu"), two) and net.buckets((3, 4), "cpu") is net.buckets((3, 4), "cpu")
    assert torch.equal(net.buckets((1, 9), "cpu"), relative_buckets((1, 9), 8)) and list(net.state_dict()) == ["table"]


def test_relative_attention_c_abi_refusals(lib):
    from pixelsplat_amd.ops import _lib
    three = C.c_int64 * 3
    s = three(96, 8, 24)
    good = dict(batch=2, heads=1, queries=6, query_start=0, grid_h=2, grid_w=3, dim=8, dtype=1, buckets=5, table_f32=0,
                scale=0.3, reserved=0, q_strides=s, k_strides=s, v_strides=s, do_strides=s, mask_stride=6)
    p = 4096          # an address that is never followed
    ok = _lib.PsRelativeAttentionDesc(**good)
    assert lib.ps_relative_attention_workspace_bytes(C.byref(ok), 0) > 0
    assert lib.ps_relative_attention_workspace_bytes(C.byref(ok), 1) > 0

    def forward(d, q=p, table=p, out=p, bias=p, ws=p, n=1 << 40):
        return lib.ps_relative_attention_forward(C.byref(d) if d else None, q, p, p, None, p, table, out, None, None, bias,
                                                 ws, n, None)

    def backward(d, stats=p, do=p, dq=p, ws=p, n=1 << 40):
        return lib.ps_relative_attention_backward(C.byref(d) if d else None, p, p, p, None, p, p, p, stats, do, dq, None,
                                                  None, None, ws, n, None)

    assert forward(None) == backward(None) == -1
    assert forward(ok, q=None) == forward(ok, q=p + 2) == forward(ok, table=None) == forward(ok, out=p + 8) == -1
    assert forward(ok, bias=None) == forward(ok, ws=None) == backward(ok, stats=None) == backward(ok, do=p + 2) == -1
    assert backward(ok, dq=p + 4) == backward(ok, ws=p + 4) == -1
    assert forward(ok, n=10) == backward(ok, n=10) == -2
    for field, value, status in [("batch", 0, -1), ("heads", -1, -1), ("queries", 0, -1), ("queries", 7, -1),
                                 ("query_start", 1, -1), ("query_start", -1, -1), ("grid_h", 0, -1), ("dim", 12, -1),
                                 ("dim", 136, -4), ("dtype", 3, -4), ("buckets", 0, -1), ("grid_w", 1024, -4),
                                 ("grid_h", 1 << 20, -4)]:
        bad = _lib.PsRelativeAttentionDesc(**{**good, field: value})
        assert forward(bad) == status and backward(bad) == status, field
        assert lib.ps_relative_attention_workspace_bytes(C.byref(bad), 1) == 0
    for more in (dict(batch=1 << 13, heads=1 << 11), dict(batch=1 << 10, heads=64, queries=1, grid_h=1, grid_w=1 << 15)):
        bad = _lib.PsRelativeAttentionDesc(**{**good, **more})
        assert forward(bad) == backward(bad) == -4, more
        assert lib.ps_relative_attention_workspace_bytes(C.byref(bad), 0) == 0
    for strides, status in [(three(96, 8, 20), -1), (three(-96, 8, 24), -1), (three(96, 8, 1 << 24), -4)]:
        assert forward(_lib.PsRelativeAttentionDesc(**{**good, "k_strides": strides})) == status
        assert backward(_lib.PsRelativeAttentionDesc(**{**good, "do_strides": strides})) == status


def test_encoder_modules_take_the_operators_when_asked(lib):
    """The options' modules and parameters; configuration objects without them (the reference's own) give the reference's."""
    from types import SimpleNamespace

    from pixelsplat_amd.encoder import (Attention, EpipolarTransformer, EpipolarTransformerCfg, FeedForward,
                                        GatedFeedForward, ImageSelfAttentionCfg)
    sa = dict(patch_size=2, num_octaves=4, num_layers=1, num_heads=2, d_token=16, d_dot=8, d_mlp=32)
    et = dict(num_octaves=10, num_layers=1, num_heads=2, num_samples=4, d_dot=8, d_mlp=32, downscale=2)
    plain = EpipolarTransformer(EpipolarTransformerCfg(self_attention=ImageSelfAttentionCfg(**sa), **et), 16, 2)
    bare = EpipolarTransformer(SimpleNamespace(self_attention=SimpleNamespace(**sa), **et), 16, 2)
    assert set(plain.state_dict()) == set(bare.state_dict())
    assert not any("relative" in n or "gate" in n for n in plain.state_dict())
    net = EpipolarTransformer(EpipolarTransformerCfg(
        self_attention=ImageSelfAttentionCfg(**sa, relative_buckets=8, gated_mlp=True, norm_groups=4), **et,
        refinement_groups=8), 16, 2)
    inner = net.transformer.layers[0][1].fn.self_attention.transformer.layers[0]
    assert isinstance(inner[1].fn, GatedFeedForward) and inner[0].fn.relative_bias.table.shape == (64, 2)
    new = set(net.state_dict()) - set(plain.state_dict())
    assert any(n.endswith("relative_bias.table") for n in new) and any(n.endswith("upscale_refinement.1.weight") for n in new)
    assert FeedForward(4, 8)(torch.zeros(2, 4)).shape == (2, 4)
    with pytest.raises(ValueError, match="self-attention"):
        Attention(8, 2, 4, selfatt=False, kv_dim=8, relative_buckets=8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        GatedFeedForward(8, 16)(torch.zeros(2, 8))


def test_group_norm_workspace_of_the_longest_samples(lib):
    """Up to 2^31 - 1 rows: the chunks' number, and with it the workspace, stays what it is at 2^30."""
    from pixelsplat_amd.ops import _lib
    for rows in ((1 << 31) - 1, (1 << 31) - 255, 2147418113):
        for dtype in (0, 1):
            size = [lib.ps_group_norm_workspace_bytes(C.byref(_lib.PsGroupNormDesc(
                samples=1, rows=r, channels=1, groups=1, dtype=dtype, activation=0, param_f32=1, eps=1e-5,
                x_sample_stride=0, x_row_stride=1, dy_sample_stride=0, dy_row_stride=1)), b) for r in (rows, 1 << 30)
                for b in (0, 1)]
            assert 0 < size[0] <= 2 * size[2] and 0 < size[1] <= 2 * size[3], (rows, size)


def test_group_norm_takes_every_number_of_groups(lib):
    """samples and channels at their limits with one channel a group: no limit of its own on their product."""
    from pixelsplat_amd.ops import _lib
    d = _lib.PsGroupNormDesc(samples=65535, rows=1, channels=8192, groups=8192, dtype=1, activation=0, param_f32=1, eps=1e-5,
                             x_sample_stride=8192, x_row_stride=8192, dy_sample_stride=8192, dy_row_stride=8192)
    # (mean, rstd)'s sums of every group at least, and of the gradient besides those of every channel
    assert lib.ps_group_norm_workspace_bytes(C.byref(d), 0) >= 16 * 65535 * 8192
    assert lib.ps_group_norm_workspace_bytes(C.byref(d), 1) >= 16 * 65535 * 8192


def test_bucket_maps_are_no_inference_tensors():
    """A map made by a validation pass is what training saves for its backward pass later."""
    from pixelsplat_amd.ops import RelativePositionBias, relative_buckets
    net = RelativePositionBias(2, 8)
    with torch.inference_mode():
        made = net.buckets((3, 4), "cpu"), relative_buckets((3, 4), 8)
    assert net.buckets((3, 4), "cpu") is made[0] and torch.equal(*made)
    for t in made:
        assert not t.is_inference()
    net.matrix((3, 4)).sum().backward()
    assert net.table.grad is not None


def test_hooks_on_the_attention_weights_see_them():
    """A hook of any kind on `attend`, or on all modules, takes the form that computes the weights (which needs no GPU)."""
    from torch.nn.modules import module as M

    from pixelsplat_amd.encoder import Attention
    net = Attention(16, 2, 8, relative_buckets=8)
    x, seen = torch.randn(1, 6, 16), []
    for add in (net.attend.register_forward_hook, net.attend.register_forward_pre_hook,
                net.attend.register_full_backward_hook, net.attend.register_full_backward_pre_hook,
                M.register_module_forward_hook, M.register_module_forward_pre_hook, M.register_module_full_backward_hook,
                M.register_module_full_backward_pre_hook):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            net(x, grid=(2, 3))
        handle = add(lambda module, *tensors: seen.append(module))
        try:
            net(x, grid=(2, 3)).sum().backward()
        finally:
            handle.remove()
        assert net.attend in seen, add
        seen.clear()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        net(x, grid=(2, 3))


def test_attention_workspace_without_the_tables_gradient(lib):
    """Where the table is frozen, nothing grows with queries times keys: 16 times the tokens take 16 times the bytes."""
    from pixelsplat_amd.ops import _lib

    def size(side, what):
        s = (C.c_int64 * 3)(side * side * 64, 64, 64)
        return lib.ps_relative_attention_workspace_bytes(C.byref(_lib.PsRelativeAttentionDesc(
            batch=2, heads=1, queries=side * side, query_start=0, grid_h=side, grid_w=side, dim=64, dtype=1, buckets=5,
            table_f32=0, scale=0.3, reserved=0, q_strides=s, k_strides=s, v_strides=s, do_strides=s, mask_stride=0)), what)

    for side in (32, 64, 128, 512):
        assert 0 < size(side, 2) <= 2 * side * side * 64 * 4 * 3 * 16 + (1 << 20), side      # parts of up to 16 splits
        assert size(side, 2) < size(side, 1)
    assert size(512, 2) <= 16 * size(128, 2) and size(512, 1) > 128 * size(128, 1)


def test_attention_backward_wants_the_workspace_of_what_it_computes(lib):
    """The size without the table's gradient is refused where that gradient is asked for."""
    from pixelsplat_amd.ops import _lib
    p, s = 4096, (C.c_int64 * 3)(96, 8, 24)          # an address that is never followed
    d = _lib.PsRelativeAttentionDesc(batch=2, heads=1, queries=6, query_start=0, grid_h=2, grid_w=3, dim=8, dtype=2, buckets=5,
                                     table_f32=0, scale=0.3, reserved=0, q_strides=s, k_strides=s, v_strides=s, do_strides=s,
                                     mask_stride=6)
    small, full = (lib.ps_relative_attention_workspace_bytes(C.byref(d), what) for what in (2, 1))
    assert 0 < small < full
    for n in (small, full - 1):
        assert lib.ps_relative_attention_backward(C.byref(d), p, p, p, None, p, p, p, p, p, p, p, p, p, p, n, None) == -2
    assert lib.ps_relative_attention_backward(C.byref(d), p, p, p, None, p, p, p, p, p, p, p, p, None, p, small - 1, None) == -2
