"""Norm of queries and keys with the rotation by position: the kernels against the formulas in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from rope_reference import angles, grid_positions, norm_rope, norm_rope_grad, rotate, rounding, STEP

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import mi355x_pisa

    return mi355x_pisa


def _rows(seed, shape, dtype, spread=1.0, layout="bthd"):
    """[B,H,T,D] values in one of the layouts a caller has."""
    b, h, t, d = shape
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)
    if layout == "bhtd":
        return x.cuda()
    if layout == "bthd":
        return x.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
    if layout == "fused":  # one part of a [B,T,3,H,D] projection
        box = torch.full((b, t, 3, h, d), math.nan, dtype=dtype, device="cuda")
        view = box[:, :, 1].permute(0, 2, 1, 3)
    else:  # rows at odd element offsets and strides
        box = torch.full((b * h * t * (d + 3) + 1,), math.nan, dtype=dtype, device="cuda")
        view = box[1:].view(b, h, t, d + 3)[..., :d]
    view.copy_(x.cuda())
    return view


def _near(actual, expected, error, what):
    off = (actual.double().cpu() - expected).abs() - rounding(actual.dtype, expected) - error * (1 + 2.0 ** -7)
    assert not torch.isnan(off).any() and float(off.max()) <= 0.0, f"{what}: {float(off.max()):.3g} over the bound"


def _turn(ops, kind, shape, axes, seed=0):
    """Rotation arguments and the reference's positions."""
    b, _, t, _ = shape
    inv = ops.rope_frequencies(axes, device="cuda")
    gen = torch.Generator().manual_seed(seed)
    if kind == "grid":
        grid = {6: (1, 2, 3), 120: (2, 6, 10), 1: (1, 1, 1), 257: (1, 257, 1), 64: (64, 1, 1)}[t]
        return {"inv_freq": inv, "axes_dims": axes, "token_grid": grid}, angles(inv, axes, grid_positions(*grid))
    if kind == "i32":
        pos = torch.randint(-50, 2 ** 30, (b, t, len(axes)), generator=gen, dtype=torch.int32)
    elif kind == "i64":
        pos = torch.randint(0, 2 ** 40, (t, len(axes)), generator=gen)
    else:
        pos = torch.rand((1, t, len(axes)), generator=gen) * 1000
    return {"inv_freq": inv, "axes_dims": axes, "positions": pos.cuda()}, angles(inv, axes, pos)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,axes,kind", [
    ((1, 1, 1, 8), (8,), "i32"),
    ((2, 3, 1, 128), (128,), "i64"),
    ((2, 5, 120, 128), (44, 42, 42), "grid"),
    ((1, 7, 257, 80), (16, 24, 24), "f32"),
    ((2, 2, 6, 256), (60, 70, 62), "grid"),
    ((1, 3, 65, 40), (10, 6, 4, 12), "i32"),
    ((3, 1, 64, 72), (2, 2, 4), "grid"),
])
def test_axial_rope(ops, dtype, interleaved, shape, axes, kind):
    turn, angle = _turn(ops, kind, shape, axes)
    for layout in ("bthd", "bhtd", "odd"):
        x = _rows(1, shape, dtype, layout=layout)
        y = ops.axial_rope(x, interleaved=interleaved, **turn)
        expected, size = rotate(x.double().cpu(), angle, interleaved)
        assert y.shape == x.shape and y.permute(0, 2, 1, 3).is_contiguous()
        _near(y, expected, 8 * STEP * size, layout)
        back = ops.axial_rope(x, interleaved=interleaved, inverse=True, **turn)
        expected, size = rotate(x.double().cpu(), -angle, interleaved)
        _near(back, expected, 8 * STEP * size, f"{layout} inverse")


NORM_CASES = [
    ((1, 1, 1, 8), 1, (8,), "i32"),
    ((2, 5, 120, 128), 5, (44, 42, 42), "grid"),
    ((1, 7, 257, 80), 3, (16, 24, 24), "f32"),
    ((2, 2, 6, 256), 6, (60, 70, 62), "grid"),
    ((1, 8, 333, 64), 2, (64,), "i64"),
    ((1, 3, 65, 168), 1, None, None),
    ((1, 4, 33, 24), 0, (8,), "i32"),
]


def _norm_call(ops, dtype, interleaved, shape, k_heads, axes, kind, weights, layout, seed=3):
    b, _, t, d = shape
    turn, angle = _turn(ops, kind, shape, axes) if axes else ({}, None)
    q = _rows(seed, shape, dtype, 2.0, layout)
    k = _rows(seed + 1, (b, k_heads, t, d), dtype, 0.5, layout) if k_heads else None
    qw = kw = None
    if weights:
        qw, kw = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(seed + i)) for i in (2, 3))
        qw, kw = qw.to(weights).cuda(), kw.to(weights).cuda() if k_heads else None
    return q, k, qw, kw, {**turn, "interleaved": interleaved, "eps": 1e-6}, angle


@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32), (F16, None)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,k_heads,axes,kind", NORM_CASES)
def test_qk_norm_rope(ops, dtype, weights, interleaved, shape, k_heads, axes, kind):
    for layout in ("bthd", "fused", "odd"):
        q, k, qw, kw, turn, angle = _norm_call(ops, dtype, interleaved, shape, k_heads, axes, kind, weights, layout)
        outs = ops.qk_norm_rope(q, k, qw, kw, **turn)
        for x, w, y in zip((q, k), (qw, kw), outs):
            if x is None:
                assert y is None
                continue
            assert y.permute(0, 2, 1, 3).is_contiguous()
            _near(y, *norm_rope(x, w, 1e-6, angle, interleaved), layout)


@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32), (F16, None)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,k_heads,axes,kind", NORM_CASES)
def test_qk_norm_rope_backward(ops, dtype, weights, interleaved, shape, k_heads, axes, kind):
    for layout in ("bthd", "odd"):
        q, k, qw, kw, turn, angle = _norm_call(ops, dtype, interleaved, shape, k_heads, axes, kind, weights, layout)
        gq = _rows(11, q.shape, dtype, 0.1, layout)
        gk = None if k is None else _rows(12, k.shape, dtype, 0.1, layout)
        grads = ops.qk_norm_rope_backward(gq, gk, q, k, qw, kw, **turn)
        for x, w, g, dx, dw in zip((q, k), (qw, kw), (gq, gk), grads[:2], grads[2:]):
            if x is None:
                assert dx is None and dw is None
                continue
            want, error, want_w, error_w = norm_rope_grad(g, x, w, 1e-6, angle, interleaved)
            _near(dx, want, error, f"{layout} dx")
            if w is None:
                assert dw is None
            else:
                _near(dw, want_w, error_w, f"{layout} dw")


def test_gradient_against_differences(ops):
    """The backward pass against central differences of the forward, both fp32 kernels.

    f is a weighted sum of the outputs; along a direction of size h its
    difference quotient is off by h^2 times a third derivative of order one and
    by the outputs' rounding over h: 1e-3 of the gradient at h = 2^-7.
    """
    shape, axes = (1, 2, 6, 64), (16, 24, 24)
    turn, _ = _turn(ops, "grid", shape, axes)
    gen = torch.Generator().manual_seed(5)
    q, k, cq, ck, uq, uk = (torch.randn(shape, generator=gen).cuda() for _ in range(6))
    w, uw = (torch.randn(64, generator=gen).cuda() for _ in range(2))

    def f(s):
        a, b = ops.qk_norm_rope(q + s * uq, k + s * uk, w + s * uw, w, **turn)
        return float(((a * cq).double().sum() + (b * ck).double().sum()).cpu())

    h = 2.0 ** -7
    dq, dk, dqw, _ = ops.qk_norm_rope_backward(cq, ck, q, k, w, w, **turn)
    along = float(((dq * uq).double().sum() + (dk * uk).double().sum() + (dqw * uw).double().sum()).cpu())
    size = float((dq * uq).double().abs().sum() + (dk * uk).double().abs().sum() + (dqw * uw).double().abs().sum())
    assert abs((f(h) - f(-h)) / (2 * h) - along) <= 1e-3 * size


def test_autograd_gives_the_backward_calls_gradients(ops):
    shape, axes = (2, 4, 120, 64), (16, 24, 24)
    turn, _ = _turn(ops, "grid", shape, axes)
    q, k = (_rows(i, shape, BF16).requires_grad_() for i in (1, 2))
    w = torch.nn.Parameter(torch.rand(64, device="cuda"))  # one weight for both: its gradients add
    a, b = ops.qk_norm_rope(q, k, w, w, **turn)
    ga, gb = torch.randn_like(a), torch.randn_like(b)
    torch.autograd.backward((a, b), (ga, gb))
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(ga, gb, q.detach(), k.detach(), w.detach(), w.detach(), **turn)
    assert torch.equal(q.grad, dq) and torch.equal(k.grad, dk) and torch.equal(w.grad, dqw + dkw)
    # only the keys' output used, its gradient expanded from one number
    q.grad = k.grad = w.grad = None
    ops.qk_norm_rope(q, k, w, w, **turn)[1].sum().backward()
    dq, dk, _, dkw = ops.qk_norm_rope_backward(torch.zeros_like(a), torch.ones_like(b), q.detach(), k.detach(),
                                               w.detach(), w.detach(), **turn)
    assert torch.equal(k.grad, dk) and torch.equal(w.grad, dkw) and not q.grad.any()
    x = _rows(3, shape, F32).requires_grad_()
    y = ops.axial_rope(x, **turn)
    g = torch.randn_like(y)
    y.backward(g)
    assert torch.equal(x.grad, ops.axial_rope(g, inverse=True, **turn))
    with torch.no_grad():
        assert not ops.axial_rope(x, **turn).requires_grad


def test_rows_of_zeros_and_values_that_are_not_finite(ops):
    """A zero row stays zero with finite gradients; an infinite or NaN row does not touch the others."""
    x = torch.randn((1, 2, 5, 64), device="cuda")
    x[0, 0, 1] = 0.0
    x[0, 1, 2, 3] = math.inf
    x[0, 1, 3, 60] = math.nan
    y, _ = ops.qk_norm_rope(x, None, eps=1e-6)
    assert not y[0, 0, 1].any()
    bad = torch.zeros((1, 2, 5), dtype=torch.bool, device="cuda")
    bad[0, 1, 2] = bad[0, 1, 3] = True
    assert torch.equal(~torch.isfinite(y).all(-1), bad)
    dx = ops.qk_norm_rope_backward(torch.ones_like(x), None, x, None, eps=1e-6)[0]
    assert torch.equal(~torch.isfinite(dx).all(-1), bad)
    # 1 / sqrt(1e-6): eps as fp32 is off by at most a step (halved by the root), root and quotient add 2.5
    assert float((dx[0, 0, 1].double() - 1000.0).abs().max()) <= 1000.0 * 4 * STEP


def test_same_bits_from_run_to_run_on_a_side_stream_and_in_a_graph(ops):
    shape, axes = (2, 6, 120, 128), (44, 42, 42)
    turn, _ = _turn(ops, "grid", shape, axes)
    q, k, gq, gk = (_rows(i, shape, BF16) for i in range(4))
    w = torch.rand(128, device="cuda")

    def call():
        return (*ops.qk_norm_rope(q, k, w, w, **turn), *ops.qk_norm_rope_backward(gq, gk, q, k, w, w, **turn),
                ops.axial_rope(q, **turn))

    eager = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for _ in range(3):
        ops.qk_norm_rope_backward(gk, gq, k, q, w, w, **turn)  # eager work between replays
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


def test_many_tokens_walked_with_the_grids_stride(ops):
    """More groups than the backward pass has workgroups, and a weight gradient of many rows."""
    shape = (2, 1, 20000, 64)
    q, g = _rows(1, shape, F32), _rows(2, shape, F32)
    pos = torch.arange(20000, device="cuda")[:, None]
    turn = {"inv_freq": ops.rope_frequencies((64,), device="cuda"), "axes_dims": (64,), "positions": pos}
    w = torch.rand(64, device="cuda")
    angle = angles(turn["inv_freq"], (64,), pos)
    _near(ops.qk_norm_rope(q, None, w, **turn)[0], *norm_rope(q, w, 1e-6, angle, False), "y")
    dx, _, dw, _ = ops.qk_norm_rope_backward(g, None, q, None, w, **turn)
    want, error, want_w, error_w = norm_rope_grad(g, q, w, 1e-6, angle, False)
    _near(dx, want, error, "dx")
    _near(dw, want_w, error_w, "dw")


def test_traces_under_compile(ops):
    shape, axes = (1, 2, 6, 64), (16, 24, 24)
    turn, _ = _turn(ops, "grid", shape, axes)
    q, k = (_rows(i, shape, BF16) for i in (1, 2))
    w = torch.rand(64, device="cuda")

    def f(q, k, w):
        a, b = ops.qk_norm_rope(q, k, w, None, **turn)
        return a.float().sum() + (ops.axial_rope(b, **turn) * 2).float().sum(), a

    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_(), w.clone().requires_grad_()]
    loss, a = f(*leaves)
    loss.backward()
    traced = [q.clone().requires_grad_(), k.clone().requires_grad_(), w.clone().requires_grad_()]
    loss_c, a_c = torch.compile(f, fullgraph=True, backend="aot_eager")(*traced)
    loss_c.backward()
    assert torch.equal(a, a_c)
    assert all(torch.equal(x.grad, y.grad) for x, y in zip(leaves, traced))


def test_refusals_on_the_device(ops):
    q = torch.zeros((1, 2, 6, 64), dtype=BF16, device="cuda")
    inv = ops.rope_frequencies((64,), device="cuda")
    pos = torch.zeros((6, 1), dtype=torch.int32, device="cuda")
    good = {"inv_freq": inv, "axes_dims": (64,), "positions": pos}
    ops.axial_rope(q, **good)
    for change, text in [
        ({"axes_dims": (32,)}, "inv_freq must be contiguous float64"),
        ({"axes_dims": (66,)}, "axes_dims"),
        ({"axes_dims": (3, 61)}, "axes_dims"),
        ({"axes_dims": (4,) * 5}, "1 to 4 axes"),
        ({"inv_freq": inv.float()}, "float64"),
        ({"inv_freq": inv.cpu()}, "on the input's device"),
        ({"positions": pos[:5]}, "positions must be"),
        ({"positions": pos.double()}, "int32, int64 or float32"),
        ({"positions": None}, "either positions or token_grid"),
        ({"token_grid": (1, 2, 3)}, "either positions or token_grid"),
        ({"positions": None, "token_grid": (1, 2, 3)}, "needs 3 axes"),
    ]:
        with pytest.raises(ValueError, match=text):
            ops.axial_rope(q, **{**good, **change})
    with pytest.raises(ValueError, match="unit stride"):
        ops.axial_rope(q.transpose(2, 3).contiguous().transpose(2, 3), **good)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.axial_rope(q[..., :20].contiguous(), **good)
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="share one dtype"):
        ops.qk_norm_rope(q, q, w, w.to(F16))
    with pytest.raises(ValueError, match="a weight must be"):
        ops.qk_norm_rope(q, q, w[:32])
    with pytest.raises(ValueError, match="k_weight needs k"):
        ops.qk_norm_rope(q, None, w, w)
    with pytest.raises(ValueError, match="eps"):
        ops.qk_norm_rope(q, q, eps=-1.0)
    with pytest.raises(ValueError, match="must share"):
        ops.qk_norm_rope(q, q[:, :, :3])
    with pytest.raises(ValueError, match="go together"):
        ops.qk_norm_rope_backward(q, None, q, q)
    with pytest.raises(ValueError, match="grad_q must be"):
        ops.qk_norm_rope_backward(q[:, :1], q, q, q)
    x = q.float().requires_grad_()
    g = torch.autograd.grad(ops.axial_rope(x, **good).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_in_place_through_the_c_abi(ops):
    """The C entry point may write its outputs over q and k."""
    from mi355x_pisa import _lib, rotary

    shape, axes = (2, 5, 120, 128), (44, 42, 42)
    turn, _ = _turn(ops, "grid", shape, axes)
    q, k = (_rows(i, shape, BF16) for i in (1, 2))
    w = torch.rand(128, device="cuda")
    want = ops.qk_norm_rope(q, k, w, w, **turn)
    rope = rotary._rope_struct(turn["inv_freq"], axes, None, turn["token_grid"], False, False)
    vq, vk = _lib.view4(q), _lib.view4(k)
    _lib.check(_lib.LIB.attn_hip_qk_norm_rope(0, 2, 2, 5, 5, 120, 128, vq, vk, vq, vk, w.data_ptr(), w.data_ptr(), 1, 1e-6,
                                              rope, _lib.stream_of(q.device)), "in place")
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("size", [1e-19, 1e-3, 1e18])
def test_rows_of_any_size_without_eps(ops, size):
    """eps = 0: the mean square of a row may lie near the ends of fp32's range (1e-38 here, where it has all its bits)."""
    x = (torch.randn((1, 2, 7, 64), generator=torch.Generator().manual_seed(1)) * size).cuda()
    _near(ops.qk_norm_rope(x, None, eps=0.0)[0], *norm_rope(x, None, 0.0, None, False), "y")


def test_many_heads_and_batches(ops):
    """Heads beyond what a tile of several tokens takes, and tiles that end inside a batch entry."""
    for shape, k_heads in (((1, 5000, 3, 8), 7), ((3, 2, 9001, 8), 1)):
        q, k = _rows(1, shape, F32), _rows(2, (shape[0], k_heads, *shape[2:]), F32)
        pos = torch.arange(shape[2], device="cuda", dtype=torch.int32)[:, None]
        turn = {"inv_freq": ops.rope_frequencies((8,), device="cuda"), "axes_dims": (8,), "positions": pos}
        angle = angles(turn["inv_freq"], (8,), pos)
        for x, y in zip((q, k), ops.qk_norm_rope(q, k, **turn)):
            _near(y, *norm_rope(x, None, 1e-6, angle, False), str(tuple(x.shape)))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape,k_heads", [((1, 3, 1025, 64), 1), ((2, 3, 1025, 128), 3), ((1, 2, 4099, 80), 1),
                                           ((3, 1, 2999, 256), 2), ((1, 40, 1031, 128), 8)])
def test_tiles_of_few_heads(ops, dtype, shape, k_heads):
    """Tiles of 2, 4, 8 and 16 tokens, the last one of a batch entry partly filled; both orders of a tile's rows."""
    for layout in ("bthd", "bhtd"):
        q, k = _rows(1, shape, dtype, layout=layout), _rows(2, (shape[0], k_heads, *shape[2:]), dtype, layout=layout)
        gq, gk = _rows(3, q.shape, dtype, layout=layout), _rows(4, k.shape, dtype, layout=layout)
        qw, kw = ((torch.rand(shape[3], generator=torch.Generator().manual_seed(i)) + 0.5).cuda() for i in (5, 6))
        pos = torch.arange(shape[2], device="cuda", dtype=torch.int32)[:, None]
        turn = {"inv_freq": ops.rope_frequencies((shape[3],), device="cuda"), "axes_dims": (shape[3],), "positions": pos}
        angle = angles(turn["inv_freq"], (shape[3],), pos)
        out = ops.qk_norm_rope(q, k, qw, kw, **turn)
        grads = ops.qk_norm_rope_backward(gq, gk, q, k, qw, kw, **turn)
        for x, w, g, y, dx, dw in zip((q, k), (qw, kw), (gq, gk), out, grads[:2], grads[2:]):
            _near(y, *norm_rope(x, w, 1e-6, angle, False), "y")
            want, error, want_w, error_w = norm_rope_grad(g, x, w, 1e-6, angle, False)
            _near(dx, want, error, "dx")
            _near(dw, want_w, error_w, "dw")
