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
    from pixelsplat_amd.ops import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(HipExtensionMissing):
        _lib.load()


def test_group_norm_refusals(lib):
    from pixelsplat_amd.ops import GroupNormAct, group_norm
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm(x, 2)
    with pytest.raises(TypeError, match="float64"):
        group_norm(x.double(), 2)
    with pytest.raises(RuntimeError, match="weight is on"):
        group_norm(_FakeGpu(x), 2, w)
    with pytest.raises(ValueError, match="activation"):
        GroupNormAct(2, 8, activation="tanh")


class _FakeGpu:
    """What check_tensors looks at of a GPU tensor."""

    def __init__(self, t):
        self.dtype, self.device, self.is_cuda, self.shape = t.dtype, torch.device("cuda:0"), True, t.shape

    def dim(self):
        return len(self.shape)


@pytest.mark.parametrize("kwargs,match", [
    (dict(num_groups=3), "do not divide"), (dict(num_groups=0), "do not divide"),
    (dict(num_groups=2, eps=-1.0), "eps"), (dict(num_groups=2, eps=float("nan")), "eps"),
    (dict(num_groups=2, activation="tanh"), "activation")])
def test_group_norm_argument_refusals(lib, kwargs, match):
    from pixelsplat_amd.ops import group_norm
    with pytest.raises(ValueError, match=match):
        group_norm(_FakeGpu(torch.zeros(2, 3, 8)), **kwargs)


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
    x, w, b = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_linear(x, w, w)
    with pytest.raises(TypeError, match="int32"):
        gated_linear(x.int(), w, w)
    fake = lambda *s, dtype=torch.float32: _FakeGpu(torch.zeros(s, dtype=dtype))  # noqa: E731
    with pytest.raises(RuntimeError, match="w_up is on"):
        gated_linear(fake(3, 8), fake(5, 8), w)
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
