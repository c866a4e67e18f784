"""Refusals of the norm and rotation entry points that need no GPU, and the frequency table."""
from __future__ import annotations

import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from mi355x_pisa import _lib

    return _lib


@pytest.fixture(scope="module")
def ops():
    import mi355x_pisa

    return mi355x_pisa


def _rope(lib, **change):
    r = lib.PisaRope()
    r.inv_freq, r.positions, r.positions_kind, r.axes = 0x1000, 0x2000, lib.POSITIONS_I32, 1
    r.axis_dims = (64, 0, 0, 0)
    for name, value in change.items():
        setattr(r, name, value)
    return r


def _forward(lib, dtype=0, weight_dtype=0, batch=1, heads=2, k_heads=2, tokens=6, dim=64, view=None, k_view=None,
             weight=0x3000, normalize=1, eps=1e-6, rope=None):
    v = lib.PisaView(0x1000, 768, 384, 64) if view is None else view
    kv = v if k_view is None else k_view
    return lib.LIB.attn_hip_qk_norm_rope(dtype, weight_dtype, batch, heads, k_heads, tokens, dim, v, kv, v, kv, weight,
                                         weight, normalize, eps, _rope(lib) if rope is None else rope, None)


@pytest.mark.parametrize("change,code,text", [
    ({"dtype": 7}, 2, "bf16, fp16 and fp32"),
    ({"weight_dtype": 1}, 2, "weights must be"),
    ({"batch": 0}, 1, "requires B>0"),
    ({"k_heads": -1}, 1, "requires B>0"),
    ({"tokens": 0}, 1, "requires B>0"),
    ({"dim": 60}, 2, "multiple of 8"),
    ({"dim": 264}, 2, "multiple of 8"),
    ({"dim": 0}, 2, "multiple of 8"),
    ({"heads": 65536}, 2, "B*H"),
    ({"eps": -1.0}, 1, "eps"),
    ({"eps": math.nan}, 1, "eps"),
    ({"eps": math.inf}, 1, "eps"),
    ({"normalize": 0}, 1, "weights need normalize"),
])
def test_forward_arguments(lib, change, code, text):
    assert _forward(lib, **change) == code
    assert text in lib.LIB.pisa_hip_last_error().decode()


@pytest.mark.parametrize("change,text", [
    ({"axes": 5}, "1 to 4 axes"),
    ({"axes": -1}, "1 to 4 axes"),
    ({"axis_dims": (0, 0, 0, 0)}, "positive even"),
    ({"axis_dims": (7, 0, 0, 0)}, "positive even"),
    ({"axis_dims": (72, 0, 0, 0)}, "positive even"),
    ({"axes": 2, "axis_dims": (40, 32, 0, 0)}, "multiple of 8 up to head_dim"),
    ({"axis_dims": (12, 0, 0, 0)}, "multiple of 8 up to head_dim"),
    ({"inv_freq": None}, "inv_freq"),
    ({"inv_freq": 0x1004}, "inv_freq"),
    ({"positions": None}, "positions"),
    ({"positions": 0x2002}, "positions"),
    ({"positions": 0x2004, "positions_kind": 2}, "positions"),
    ({"positions_kind": 9}, "positions kind"),
    ({"positions_kind": -1}, "positions kind"),
    ({"positions_kind": 0}, "3 axes"),
])
def test_rotation_arguments(lib, change, text):
    assert _forward(lib, rope=_rope(lib, **change)) == 1
    assert text in lib.LIB.pisa_hip_last_error().decode()


@pytest.mark.parametrize("grid", [(1, 2, 4), (0, 2, 3), (-1, -2, 3), (1, 65536, 65536)])
def test_grid_must_hold_the_tokens(lib, grid):
    rope = _rope(lib, positions_kind=0, axes=3, axis_dims=(16, 24, 24, 0), grid=lib.grid(*grid))
    assert _forward(lib, rope=rope) == 1
    assert "does not match 6 tokens" in lib.LIB.pisa_hip_last_error().decode()


def test_views_must_be_there_and_aligned_to_their_element(lib):
    assert _forward(lib, view=lib.PisaView(None, 0, 0, 0)) == 1
    assert _forward(lib, view=lib.PisaView(0x1001, 768, 384, 64)) == 1
    assert _forward(lib, k_view=lib.PisaView(None, 0, 0, 0)) == 1
    assert "k must be" in lib.LIB.pisa_hip_last_error().decode()


def test_backward_workspace(lib):
    size = lib.LIB.attn_hip_qk_norm_rope_backward_workspace_bytes
    assert size(128, 0) == 0 and size(0, 1) == 0 and size(257, 1) == 0
    assert size(128, 1) == 2 * 128 * 1024 * 4
    v = lib.PisaView(0x1000, 768, 384, 64)

    def call(workspace, held):
        return lib.LIB.attn_hip_qk_norm_rope_backward(0, 0, 1, 2, 2, 6, 64, v, v, v, v, 0x3000, 0x3000, v, v, 0x4000, 0x4000,
                                                      1e-6, _rope(lib), workspace, held, None)

    assert call(None, 1 << 30) == 3 and call(0x5008, 1 << 30) == 3 and call(0x5000, size(64, 1) - 1) == 3
    assert "workspace" in lib.LIB.pisa_hip_last_error().decode()


def test_python_refusals_without_a_device(ops):
    x = torch.zeros((1, 2, 6, 64), dtype=torch.bfloat16)
    inv = ops.rope_frequencies((64,))
    with pytest.raises(TypeError):
        ops.qk_norm_rope([1.0], x)
    with pytest.raises(ValueError, match="B,H,T,D"):
        ops.qk_norm_rope(x[0], x[0])
    with pytest.raises(ValueError, match="every dimension positive"):
        ops.axial_rope(x[:, :, :0], inv, (64,), torch.zeros((0, 1)))
    with pytest.raises(ValueError, match="ROCm device"):
        ops.qk_norm_rope(x, x)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.axial_rope(x, inv, (64,), torch.zeros((6, 1)))


def test_frequencies(ops):
    f = ops.rope_frequencies((4, 6), theta=(100.0, 8.0))
    assert f.dtype == torch.float64
    want = torch.tensor([1.0, 0.1, 1.0, 0.5, 0.25], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-15, atol=0)
    for bad in ((), (3,), (0, 4), (-2,)):
        with pytest.raises(ValueError, match="axes_dims"):
            ops.rope_frequencies(bad)
    for theta in (0.0, -1.0, math.inf, (1.0,)):
        with pytest.raises(ValueError, match="theta"):
            ops.rope_frequencies((4, 6), theta=theta)
