"""Exact attention for training: the forward with log sums and the backward pass against 64-bit formulas."""
from __future__ import annotations

import math

import pytest
import torch

from attention_reference import near, reference

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    import mi355x_pisa

    return mi355x_pisa


def _rows(seed, shape, dtype, spread=1.0, layout="bthd"):
    b, h, t, d = shape
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()
    if layout == "bhtd":
        return x
    if layout == "fused":  # one part of a [B,T,3,H,D] projection
        box = torch.full((b, t, 3, h, d), math.nan, dtype=dtype, device="cuda")
        view = box[:, :, 1].permute(0, 2, 1, 3)
    else:
        view = torch.empty((b, t, h, d), dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    return view.copy_(x)


def _inputs(dtype, shape, layout="bthd", spread=1.0, grad_spread=1.0, seed=0):
    b, h, hk, tq, tk, d = shape
    q = _rows(seed + 1, (b, h, tq, d), dtype, spread, layout)
    k = _rows(seed + 2, (b, hk, tk, d), dtype, spread, layout)
    v = _rows(seed + 3, (b, hk, tk, d), dtype, 1.0, layout)
    g = _rows(seed + 4, (b, h, tq, d), dtype, grad_spread, layout)
    return q, k, v, g


def _lengths(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def _check(ops, q, k, v, g, scale, lengths=None, grad_lse=None):
    out, lse = ops.dense_attention_with_lse(q, k, v, scale, kv_lengths=lengths)
    grads = ops.dense_attention_backward(g, q, k, v, out, lse, scale, kv_lengths=lengths, grad_lse=grad_lse)
    want = reference(q, k, v, scale, lengths, g, grad_lse)
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        near(x, want[name], name)
        if name != "lse":
            assert x.permute(0, 2, 1, 3).is_contiguous()
    return (out, lse, *grads)


CASES = [
    # B, H, Hkv, Tq, Tk, D, lengths
    ((1, 1, 1, 1, 1, 8), None),
    ((1, 2, 2, 64, 64, 64), None),
    ((2, 4, 2, 65, 129, 128), [129, 0]),
    ((1, 3, 1, 257, 31, 40), None),
    ((1, 2, 2, 300, 300, 80), None),
    ((2, 2, 1, 33, 200, 96), [1, 200]),
    ((1, 1, 1, 130, 70, 160), None),
    ((1, 2, 1, 70, 130, 192), [95]),
    ((1, 1, 1, 100, 161, 256), None),
    ((3, 2, 2, 1, 300, 128), [0, 5, 300]),
    ((1, 2, 2, 1000, 700, 64), [-7]),       # counts outside [0, Tk] are taken into it
    ((1, 2, 2, 513, 700, 128), [100000]),
    ((1, 1, 1, 2500, 40, 128), None),       # few keys: the queries are split over workgroups
    ((1, 4, 1, 40, 2500, 72), None),        # few queries: the keys are split
    ((4, 64, 64, 65, 65, 64), None),        # as many workgroups as CUs: no split
    ((1, 1, 1, 640, 640, 128), None),
    ((2, 2, 2, 65, 900, 160), [70, 833]),   # waves that share a query block, some of them without a key
    ((3, 1, 1, 40, 1000, 256), [0, 64, 1000]),
    ((4, 2, 1, 100, 1100, 64), [1, 129, 0, 1024]),
    ((2, 2, 1, 70, 1500, 96), [1500, 333]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,lengths", CASES)
def test_against_the_formulas(ops, dtype, shape, lengths):
    _check(ops, *_inputs(dtype, shape), shape[5] ** -0.5, _lengths(lengths))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["bhtd", "fused"])
def test_layouts(ops, dtype, layout):
    _check(ops, *_inputs(dtype, (2, 3, 3, 100, 170, 128), layout), 0.1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_peaked_rows_and_large_scores(ops, dtype, dim):
    """Rows that one key holds almost alone."""
    _check(ops, *_inputs(dtype, (1, 2, 2, 200, 333, dim), spread=4.0), 0.5)


@pytest.mark.parametrize("dtype,grad_spread", [(F16, 2.0 ** -12), (F16, 256.0), (BF16, 1e-20), (BF16, 1e15)])
def test_small_and_large_gradients(ops, dtype, grad_spread):
    """Gradients near the ends of fp16's range keep their bits in the products (dq and dk themselves are rounded to it)."""
    _check(ops, *_inputs(dtype, (1, 2, 1, 300, 700, 64), grad_spread=grad_spread), 0.125)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [None, [77, 0]])
def test_gradient_of_the_log_sums(ops, dtype, lengths):
    q, k, v, g = _inputs(dtype, (2, 4, 2, 90, 150, 64))
    dl = torch.randn((2, 4, 90), generator=torch.Generator().manual_seed(9)).cuda() * 3
    _check(ops, q, k, v, g, 0.125, _lengths(lengths), dl)
    _check(ops, q, k, v, torch.zeros_like(g), 0.125, _lengths(lengths), dl)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_masked_keys_may_hold_anything(ops, dtype):
    q, k, v, g = _inputs(dtype, (2, 2, 2, 70, 200, 128))
    lengths = _lengths([130, 64])
    want = _check(ops, q, k, v, g, 0.1, lengths)
    for b, n in enumerate((130, 64)):
        k[b, :, n:], v[b, :, n:] = math.nan, math.inf
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.1, kv_lengths=lengths)
    got = (out, lse, *ops.dense_attention_backward(g, q, k, v, out, lse, 0.1, kv_lengths=lengths))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[3][1, :, 64:].any() and not got[4][1, :, 64:].any()


def test_no_key_at_all(ops):
    q, k, v, g = _inputs(BF16, (1, 2, 2, 70, 200, 128))
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.1, kv_lengths=_lengths([0]))
    assert not out.any() and torch.equal(lse, torch.full_like(lse, -math.inf))
    assert not any(x.any() for x in ops.dense_attention_backward(g, q, k, v, out, lse, 0.1, kv_lengths=_lengths([0])))


def test_zero_gradients_in_fp16(ops):
    q, k, v, g = _inputs(F16, (1, 2, 2, 70, 200, 64))
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.125)
    assert not any(x.any() for x in ops.dense_attention_backward(torch.zeros_like(g), q, k, v, out, lse, 0.125))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_row_that_is_not_finite_leaves_the_other_heads_alone(ops, dtype):
    q, k, v, g = _inputs(dtype, (1, 3, 3, 130, 100, 64))
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.125)
    want = ops.dense_attention_backward(g, q, k, v, out, lse, 0.125)
    g = g.clone()
    g[0, 1, 7, 3] = math.nan
    got = ops.dense_attention_backward(g, q, k, v, out, lse, 0.125)
    for a, b in zip(got, want):
        assert torch.equal(a[:, 0::2], b[:, 0::2])
    assert torch.isnan(got[0][0, 1, 7]).all() and torch.isnan(got[2][0, 1, :, 3]).all()


def test_gradients_against_differences(ops):
    """The backward pass against central differences of a 64-bit forward.

    With inputs rounded to bf16 the formulas' gradient is exact up to the
    bound of test_against_the_formulas; a step of 2^-10 along a random direction
    leaves 2^-20 times a third derivative of order one.
    """
    q, k, v, g = _inputs(BF16, (1, 2, 1, 20, 50, 64))
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.125)
    grads = ops.dense_attention_backward(g, q, k, v, out, lse, 0.125)
    want = reference(q, k, v, 0.125, None, g)
    gen = torch.Generator().manual_seed(3)
    along = [torch.randn(x.shape, generator=gen, dtype=torch.float64) for x in (q, k, v)]

    def f(step):
        a, b, c = (x.double().cpu() + step * y for x, y in zip((q, k, v), along))
        s = 0.125 * a @ b.repeat_interleave(2, 1).transpose(2, 3)
        return float((torch.softmax(s, -1) @ c.repeat_interleave(2, 1) * g.double().cpu()).sum())

    h = 2.0 ** -10
    slope = (f(h) - f(-h)) / (2 * h)
    got = sum(float((x.double().cpu() * y).sum()) for x, y in zip(grads, along))
    error = sum(float((want[n][1] * y.abs()).sum()) for n, y in zip(("dq", "dk", "dv"), along))
    size = sum(float((want[n][0] * y).abs().sum()) for n, y in zip(("dq", "dk", "dv"), along))
    assert abs(slope - got) <= error + 1e-4 * size


def test_autograd(ops):
    q, k, v, g = _inputs(BF16, (2, 4, 2, 90, 150, 64))
    lengths = _lengths([150, 33])
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.125, kv_lengths=lengths)
    dl = torch.randn_like(lse)
    want = ops.dense_attention_backward(g, q, k, v, out, lse, 0.125, kv_lengths=lengths, grad_lse=dl)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o, l = ops.dense_attention_with_lse(*leaves, 0.125, kv_lengths=lengths)
    assert torch.equal(o, out) and torch.equal(l, lse)
    for got, x in zip(torch.autograd.grad((o, l), leaves, (g, dl), retain_graph=True), want):
        assert torch.equal(got, x)
    # one output alone, an expanded gradient, one frozen side
    zero = torch.zeros_like(g)
    got = torch.autograd.grad(l.sum(), leaves, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.dense_attention_backward(
        zero, q, k, v, out, lse, 0.125, kv_lengths=lengths, grad_lse=torch.ones_like(lse))))
    ones = ops.dense_attention_backward(torch.ones_like(g), q, k, v, out, lse, 0.125, kv_lengths=lengths)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o.sum(), leaves), ones))
    o, _ = ops.dense_attention_with_lse(leaves[0], k, v, 0.125, kv_lengths=lengths)
    assert torch.equal(torch.autograd.grad(o.sum(), leaves[0])[0], ones[0])
    o, _ = ops.dense_attention_with_lse(q, leaves[1], v, 0.125, kv_lengths=lengths)
    assert torch.equal(torch.autograd.grad(o.sum(), leaves[1])[0], ones[1])
    x = q.clone().requires_grad_()
    first = torch.autograd.grad(ops.dense_attention_with_lse(x, k, v, 0.125)[0].float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        first.sum().backward()


def test_the_output_is_dense_attentions(ops):
    """Same operator as dense_attention, which divides by the sum of the rounded probabilities: one more u |out|."""
    q, k, v, _ = _inputs(BF16, (2, 4, 4, 500, 700, 128))
    out, _ = ops.dense_attention_with_lse(q, k, v, 0.1)
    other = ops.dense_attention(q, k, v, 0.1)
    _, error = reference(q, k, v, 0.1)["out"]
    assert bool(((out.double() - other.double()).abs().cpu() <= 3 * error * (1 + 2.0 ** -6)).all())


def test_same_bits_on_a_side_stream_and_in_graphs_that_live_together(ops):
    """Run to run, on another stream, and replayed from two graphs captured one after the other."""
    q, k, v, g = _inputs(BF16, (1, 4, 2, 300, 900, 128))
    lengths = _lengths([850])

    def call(scale):
        out, lse = ops.dense_attention_with_lse(q, k, v, scale, kv_lengths=lengths)
        return (out, lse, *ops.dense_attention_backward(g, q, k, v, out, lse, scale, kv_lengths=lengths))

    eager = [call(0.1), call(0.2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call(0.1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager[0], again))
    graphs, captured = [], []
    for scale in (0.1, 0.2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(call(scale))
        graphs.append(graph)
    for _ in range(3):
        call(0.3)  # eager work between replays
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for want, got in zip(eager, captured):
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    # what a replay reads at its time: a new count of keys
    lengths.fill_(64)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured[0], call(0.1)))


def test_traces_under_compile(ops):
    q, k, v, g = _inputs(BF16, (1, 2, 1, 90, 150, 64))

    def f(q, k, v):
        out, lse = ops.dense_attention_with_lse(q, k, v, 0.125)
        return (out.float() * g.float()).sum() + lse.sum(), out

    plain, traced = ([x.clone().requires_grad_() for x in (q, k, v)] for _ in range(2))
    loss, out = f(*plain)
    loss.backward()
    loss_c, out_c = torch.compile(f, fullgraph=True, backend="aot_eager")(*traced)
    loss_c.backward()
    assert torch.equal(out, out_c) and all(torch.equal(a.grad, b.grad) for a, b in zip(plain, traced))


def test_norm_rotation_attention_and_back(ops):
    """A layer as it is trained: qkv -> norm and rotation -> attention, back to the projection and the norms' weights."""
    b, t, h, d, grid, axes = 2, 120, 4, 64, (2, 6, 10), (16, 24, 24)
    gen = torch.Generator().manual_seed(1)
    qkv = (torch.randn((b, t, 3, h, d), generator=gen)).to(BF16).cuda().requires_grad_()
    qw, kw = (torch.nn.Parameter((1 + 0.2 * torch.randn(d, generator=gen)).cuda()) for _ in range(2))
    g = torch.randn((b, t, h * d), generator=gen).to(BF16).cuda()
    inv = ops.rope_frequencies(axes, device="cuda")
    q, k, v = (qkv[:, :, i].permute(0, 2, 1, 3) for i in range(3))
    qn, kn = ops.qk_norm_rope(q, k, qw, kw, inv_freq=inv, axes_dims=axes, token_grid=grid)
    out, _ = ops.dense_attention_with_lse(qn, kn, v, d ** -0.5)
    out.permute(0, 2, 1, 3).reshape(b, t, h * d).backward(g)
    # the same chain of plain calls
    with torch.no_grad():
        o, lse = ops.dense_attention_with_lse(qn, kn, v, d ** -0.5)
        g4 = g.view(b, t, h, d).permute(0, 2, 1, 3)
        dqn, dkn, dv = ops.dense_attention_backward(g4, qn, kn, v, o, lse, d ** -0.5)
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(dqn, dkn, q, k, qw, kw, inv_freq=inv, axes_dims=axes, token_grid=grid)
        want = torch.stack([x.permute(0, 2, 1, 3) for x in (dq, dk, dv)], dim=2)
    assert torch.equal(qkv.grad, want) and torch.equal(qw.grad, dqw) and torch.equal(kw.grad, dkw)
    # and the whole layer in 64 bits: three roundings to bf16 lie in a row on the way (P and dS, the normed q and k,
    # the gradients between the steps), each 2^-8 of its terms; 3 % of a tensor's norm is eight times that
    leaf = [x.detach().double().cpu().requires_grad_() for x in (qkv, qw, kw)]
    from rope_reference import angles, grid_positions

    angle = angles(inv, axes, grid_positions(*grid))

    def turned(x, w):
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        half = d // 2
        a, c, s = n[..., :half], angle.cos(), angle.sin()
        e = n[..., half:]
        return torch.cat((a * c - e * s, a * s + e * c), dim=-1)

    x = [leaf[0][:, :, i].permute(0, 2, 1, 3) for i in range(3)]
    z = torch.softmax(turned(x[0], leaf[1]) @ turned(x[1], leaf[2]).transpose(2, 3) * d ** -0.5, -1) @ x[2]
    exact = torch.autograd.grad(z, leaf, g4.double().cpu())
    for got, e in zip((qkv.grad, qw.grad, kw.grad), exact):
        assert float((got.double().cpu() - e).norm() / e.norm()) < 0.03


def test_refusals_on_the_device(ops):
    q, k, v, g = _inputs(BF16, (2, 4, 2, 9, 12, 64))
    out, lse = ops.dense_attention_with_lse(q, k, v, 0.125)

    def refused(error, text, *args, **kwargs):
        with pytest.raises(error, match=text):
            ops.dense_attention_with_lse(*args, **kwargs)

    refused(ValueError, "do not divide", q[:, :3], k, v, 0.1)
    refused(ValueError, "must match", q, k, v[:, :, :5], 0.1)
    refused(ValueError, "share batch", q, k[:1], v[:1], 0.1)
    refused(ValueError, "one dtype", q, k, v.half(), 0.1)
    refused(ValueError, "one dtype", q.float(), k.float(), v.float(), 0.1)
    refused(ValueError, "unit stride", q, k.transpose(2, 3).contiguous().transpose(2, 3), v, 0.1)
    refused(ValueError, "scale", q, k, v, 0.0)
    refused(ValueError, "scale", q, k, v, math.nan)
    refused(ValueError, "every dimension", q, k[:, :, :0], v[:, :, :0], 0.1)
    refused(ValueError, "kv_lengths", q, k, v, 0.1, kv_lengths=torch.ones(2, device="cuda"))
    refused(ValueError, "kv_lengths", q, k, v, 0.1, kv_lengths=_lengths([1, 2, 3]))
    refused(ValueError, "kv_lengths", q, k, v, 0.1, kv_lengths=_lengths([1, 2]).cpu())
    refused(TypeError, "kv_lengths", q, k, v, 0.1, kv_lengths=[1, 2])
    wide = torch.zeros((1, 1, 4, 68), dtype=BF16, device="cuda")
    refused(RuntimeError, "multiple of 8", wide, wide, wide, 0.1)
    odd = torch.zeros(2 * 9 * 64 + 1, dtype=BF16, device="cuda")[1:].view(1, 2, 9, 64)
    refused(RuntimeError, "16-byte aligned", odd, odd, odd, 0.1)

    def refused_back(error, text, **change):
        args = {"grad_out": g, "q": q, "k": k, "v": v, "out": out, "lse": lse, "scale": 0.125, **change}
        with pytest.raises(error, match=text):
            ops.dense_attention_backward(**args)

    refused_back(ValueError, "grad_out must be", grad_out=g[:, :, :3])
    refused_back(ValueError, "out must be", out=out.half())
    refused_back(ValueError, "lse must be", lse=lse.double())
    refused_back(ValueError, "lse must be", lse=lse[:, :, :4])
    refused_back(ValueError, "grad_lse must be", grad_lse=lse[:1])
    refused_back(TypeError, "lse must be", lse=None)
    refused_back(TypeError, "grad_out must be", grad_out=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,lengths,split", [
    ((1, 8, 8, 1, 9216, 128), None, True),
    ((2, 3, 1, 1, 8369, 72), [8369, 70], True),  # entry 1: most parts without a key
    ((1, 4, 2, 130, 4100, 64), None, False),       # eight waves a block without a join are as fast
    ((2, 2, 2, 2, 3400, 40), [0, 3399], False),
    ((1, 4, 2, 130, 8100, 64), None, True),
    ((2, 2, 2, 2, 7000, 40), [0, 6999], True),     # entry 0: every part without a key
    ((1, 3, 3, 65, 2999, 160), None, True),
    ((2, 1, 1, 40, 2500, 256), [65, 2500], True),
    ((1, 16, 4, 7, 5000, 192), [4990], True),
])
def test_few_queries_against_long_key_lists(ops, dtype, shape, lengths, split):
    """A query block shared by several workgroups and joined."""
    import mi355x_pisa._lib as lib

    b, h, hk, tq, tk, d = shape
    size = lib.LIB.attn_hip_dense_forward_lse_workspace_bytes
    packed = lib.LIB.attn_hip_dense_workspace_bytes(b, hk, tk, d)
    assert (size(0, b, h, hk, tq, tk, d) > packed + 2 * b * h * 64 * d * 4) == split  # two parts at least
    assert size(0, b, h, hk, 9216, tk, d) == packed
    call = _inputs(dtype, shape)
    first = _check(ops, *call, shape[5] ** -0.5, _lengths(lengths))
    out, lse = ops.dense_attention_with_lse(*call[:3], shape[5] ** -0.5, kv_lengths=_lengths(lengths))
    assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_shared_query_blocks_replay_in_a_graph(ops):
    q, k, v, _ = _inputs(BF16, (1, 4, 2, 3, 4000, 128))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            want = ops.dense_attention_with_lse(q, k, v, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.dense_attention_with_lse(q, k, v, 0.1)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        k.mul_(-1 - i)  # eager work between the replays
        want = ops.dense_attention_with_lse(q, k, v, 0.1)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["bthd", "bhtd", "fused"])
@pytest.mark.parametrize("shape,lengths", [
    ((2, 4, 2, 65, 129, 64), [129, 0]),
    ((2, 4, 2, 65, 129, 128), [1, 64]),
    ((1, 6, 3, 130, 300, 72), [299]),
    ((1, 8, 8, 200, 1000, 40), None),
    ((3, 2, 1, 1, 500, 104), [500, 63, 65]),
])
def test_small_calls_in_place(ops, dtype, layout, shape, lengths):
    """Keys and values read where they are: NaN beside every row (fused) and in masked keys."""
    q, k, v, g = _inputs(dtype, shape, layout)
    if lengths is not None:
        for i, n in enumerate(lengths):
            k[i, :, n:] = math.nan
            v[i, :, n:] = math.inf
    _check(ops, q, k, v, g, shape[5] ** -0.5, _lengths(lengths))
