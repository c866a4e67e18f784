"""Refusals and workspace sizes of the training entry points that need no GPU."""
from __future__ import annotations

import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from mi355x_pisa import _lib

    return _lib


def _view(lib, ptr=0x10000):
    return lib.PisaView(ptr, 4096, 1024, 128)


BIG = 1 << 40


def _forward(lib, dtype=0, batch=1, heads=4, kv_heads=2, q_tokens=6, kv_tokens=9, dim=64, view=None, lse=0x20000,
             lengths=None, scale=0.1, workspace=0x30000, held=BIG):
    v = _view(lib)
    x = v if view is None else view
    return lib.LIB.attn_hip_dense_forward_lse(dtype, batch, heads, kv_heads, q_tokens, kv_tokens, dim, x, v, v, v, lse,
                                              lengths, scale, workspace, held, None)


def _backward(lib, dtype=0, batch=1, heads=4, kv_heads=2, q_tokens=6, kv_tokens=9, dim=64, view=None, lse=0x20000,
              grad_lse=None, lengths=None, scale=0.1, dq="view", dk="view", dv="view", workspace=0x30000, held=BIG):
    v = _view(lib)
    x = v if view is None else view
    outs = [v if t == "view" else t for t in (dq, dk, dv)]
    return lib.LIB.attn_hip_dense_backward(dtype, batch, heads, kv_heads, q_tokens, kv_tokens, dim, v, v, v, v, x, lse,
                                           grad_lse, lengths, scale, *outs, workspace, held, None)


SHARED = [
    ({"dtype": 2}, 2, "bf16 and fp16 only"),
    ({"batch": 0}, 1, "requires B>0"),
    ({"kv_heads": 0}, 1, "requires B>0"),
    ({"q_tokens": 0}, 1, "requires B>0"),
    ({"kv_tokens": -1}, 1, "requires B>0"),
    ({"kv_heads": 3}, 1, "do not divide"),
    ({"heads": 65536}, 2, "B*H"),
    ({"dim": 60}, 2, "multiple of 8"),
    ({"dim": 264}, 2, "multiple of 8"),
    ({"scale": 0.0}, 1, "scale"),
    ({"scale": math.nan}, 1, "scale"),
    ({"scale": math.inf}, 1, "scale"),
    ({"lengths": 0x2001}, 1, "kv_lengths"),
    ({"kv_tokens": 1 << 24, "dim": 256, "heads": 2, "q_tokens": 1}, 2, "above 2 GiB"),
    ({"lse": None}, 1, "lse"),
    ({"lse": 0x2002}, 1, "lse"),
    ({"workspace": None}, 3, "workspace"),
    ({"workspace": 0x30008}, 3, "workspace"),
    ({"held": 100}, 3, "workspace"),
]


@pytest.mark.parametrize("change,code,text", SHARED)
@pytest.mark.parametrize("call", [_forward, _backward])
def test_arguments(lib, call, change, code, text):
    assert call(lib, **change) == code
    assert text in lib.LIB.pisa_hip_last_error().decode()


@pytest.mark.parametrize("call", [_forward, _backward])
def test_views_must_be_aligned(lib, call):
    for bad in (lib.PisaView(None, 0, 0, 0), _view(lib, 0x10008), lib.PisaView(0x10000, 4096, 1024, 100)):
        assert call(lib, view=bad) == 1


def test_backward_outputs(lib):
    none = lib.PisaView(None, 0, 0, 0)
    assert _backward(lib, dq=none, dk=none, dv=none) == 1 and "must be given" in lib.LIB.pisa_hip_last_error().decode()
    assert _backward(lib, dk=none) == 1 and "go together" in lib.LIB.pisa_hip_last_error().decode()
    assert _backward(lib, dq=_view(lib, 0x10008)) == 1
    assert _backward(lib, grad_lse=0x2002) == 1


def test_workspace_bytes(lib):
    size = lib.LIB.attn_hip_dense_backward_workspace_bytes
    assert size(2, 1, 4, 2, 6, 9, 64) == 0 and size(0, 1, 4, 3, 6, 9, 64) == 0 and size(0, 1, 4, 2, 6, 9, 4) == 0
    # 32 rows of two operands (Q and dO, or K and V) and 1 KB, of which 256 bytes are the rows' values
    unit = 2 * 64 * 32 * 2 + 1024
    assert size(0, 1, 4, 2, 64, 64, 64) == 4 * 2 * unit + 2 * 2 * unit
    # fp16 keeps the largest row norms by block too
    assert size(1, 1, 4, 2, 64, 64, 64) == size(0, 1, 4, 2, 64, 64, 64) + 3 * 256
    # many workgroups: no parts; few: fp32 parts of the gradients
    whole = size(0, 4, 64, 64, 128, 128, 128)
    unit = 2 * 128 * 32 * 2 + 1024
    assert whole == 256 * 4 * (unit + unit)
    assert size(0, 1, 1, 1, 4096, 64, 128) > 128 * unit + 2 * unit + 2 * 64 * 128 * 4


def test_forward_workspace_bytes(lib):
    size, packed = lib.LIB.attn_hip_dense_forward_lse_workspace_bytes, lib.LIB.attn_hip_dense_workspace_bytes
    assert size(2, 1, 4, 2, 6, 9, 64) == 0 and size(0, 1, 4, 3, 6, 9, 64) == 0 and size(0, 1, 4, 2, 6, 9, 4) == 0
    assert size(0, 2, 16, 4, 9216, 512, 128) == packed(2, 4, 512, 128)
    assert size(0, 1, 300, 300, 1, 9216, 128) == packed(1, 300, 9216, 128)  # as many query blocks as CUs: not shared
    # a query block shared by several workgroups: 64 rows of 128 dims and a log sum each
    parts, rest = divmod(size(0, 1, 1, 1, 64, 9216, 128) - packed(1, 1, 9216, 128), 64 * 128 * 4 + 64 * 4)
    assert 2 <= parts <= 32 and rest == 0
    need = size(1, 1, 1, 1, 64, 9216, 128)
    assert _forward(lib, dtype=1, heads=1, kv_heads=1, q_tokens=64, kv_tokens=9216, dim=128, held=need - 1) == 3
    assert b"workspace" in lib.LIB.pisa_hip_last_error()


def test_capabilities_name_the_training_calls():
    import mi355x_pisa as ops

    caps = ops.capabilities()
    assert caps["dense_training_dtypes"] == (torch.bfloat16, torch.float16)
    assert caps["dense_training_head_dims"] == caps["rope_head_dims"] == tuple(range(8, 257, 8))
    assert caps["rope_dtypes"] == (torch.bfloat16, torch.float16, torch.float32)
    assert caps["backward"] is False  # PISA's


def test_python_refusals_without_a_device():
    import mi355x_pisa as ops

    x = torch.zeros((1, 2, 6, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.dense_attention_with_lse(x, None, x, 0.1)
    with pytest.raises(ValueError, match="B,H,T,D"):
        ops.dense_attention_with_lse(x[0], x, x, 0.1)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.dense_attention_with_lse(x, x, x, 0.1)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.dense_attention_backward(x, x, x, x, x, torch.zeros((1, 2, 6)), 0.1)
