"""The training and position operators around the attention kernels, as measurable cases.

* ``rope``  - mi355x_pisa.axial_rope: rotary positions with several axes;
* ``norm``  - mi355x_pisa.qk_norm_rope: RMS norm of queries and keys for each
  head with the rotation in the same pass; with ``grad`` also
  mi355x_pisa.qk_norm_rope_backward;
* ``train`` - mi355x_pisa.dense_attention_with_lse followed by
  mi355x_pisa.dense_attention_backward: one attention layer of a training step.
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_THETA = 10000.0


# ------------------------------------------------------------------ cases
def _rope(dtype, batch, heads, tokens, dim, axes, positions, interleaved, frames=0, height=0, width=0, **name):
    return {**name, "kind": "rope", "dtype": dtype, "batch": batch, "heads": heads, "tokens": tokens, "dim": dim,
            "axes": axes, "positions": positions, "interleaved": interleaved, "frames": frames, "height": height,
            "width": width}


def _norm(dtype, batch, heads, k_heads, tokens, dim, axes, positions, interleaved, grad, fused=False, frames=0,
          height=0, width=0, **name):
    return {**name, "kind": "norm", "dtype": dtype, "batch": batch, "heads": heads, "k_heads": k_heads,
            "tokens": tokens, "dim": dim, "axes": axes, "positions": positions, "interleaved": interleaved,
            "grad": grad, "fused_qkv": fused, "frames": frames, "height": height, "width": width}


def _train(dtype, batch, heads, kv_heads, tokens, kv_tokens, dim, lengths=False, **name):
    return {**name, "kind": "train", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "tokens": tokens, "kv_tokens": kv_tokens, "dim": dim, "lengths": lengths}


def listed():
    return [
        # one new token of each of four sequences, far along: launch and host time
        _rope("fp16", 4, 16, 1, 128, "128", "int", False, name="rope-token"),
        # fractional positions, odd length, part of the dims rotated, full precision
        _rope("fp32", 2, 10, 4001, 80, "16,24,24", "float", False, name="rope-fp32"),
        # video tokens (16 x 32 x 64), adjacent pairs
        _rope("bf16", 1, 40, 32768, 128, "44,42,42", "grid", True, 16, 32, 64, name="rope-video"),
        # a 96 x 96 token image, both guidance halves, before its attention
        _norm("bf16", 2, 16, 16, 9216, 128, "44,42,42", "grid", False, False, frames=1, height=96, width=96,
              name="norm-image"),
        # queries and keys read in place from one fused projection
        _norm("bf16", 1, 56, 56, 9170, 128, "32,48,48", "int", True, False, fused=True, name="norm-fused-qkv"),
        # a short training step with few shared key heads
        _norm("fp16", 1, 8, 2, 333, 64, "16,24,24", "int", True, True, name="norm-grad-small"),
        # the image layer's training step
        _norm("bf16", 2, 16, 16, 9216, 128, "44,42,42", "grid", False, True, frames=1, height=96, width=96,
              name="norm-grad-image"),
        # a low-resolution stage: few heads and an odd length
        _train("fp16", 1, 8, 8, 1000, 1000, 64, name="train-small"),
        # a wide head
        _train("fp16", 2, 8, 8, 1024, 1024, 160, name="train-wide"),
        # image tokens against text of up to 512 tokens, a length for each batch entry
        _train("bf16", 2, 16, 16, 9216, 512, 128, lengths=True, name="train-cross"),
        # four query heads to a key head, an odd length
        _train("bf16", 1, 16, 4, 4001, 4001, 128, name="train-grouped"),
        # self-attention of the 96 x 96 image, both guidance halves
        _train("bf16", 2, 16, 16, 9216, 9216, 128, name="train-image"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _split_axes(rng, rotated, count):
    """`rotated` dims (a multiple of 8) split over `count` axes, each an even number."""
    pairs, dims = rotated // 2, []
    for left in range(count - 1, 0, -1):
        take = rng.randint(1, pairs - left)
        dims.append(2 * take)
        pairs -= take
    return ",".join(map(str, dims + [2 * pairs]))


def draw(rng):
    """One more case of the ranges above, at most as large as the largest listed one of its kind."""
    kind = rng.choice(("rope", "norm", "norm", "train", "train", "train"))
    dtype = rng.choice(("bf16", "fp16"))
    if kind == "train":
        dim = rng.choice((64, 128, 128, 8 * rng.randint(2, 32)))
        kv_heads, group = rng.randint(1, 16), rng.choice((1, 1, 1, 2, 4))
        batch = rng.randint(1, 3)
        tokens = _log_int(rng, 1, 9216)
        kv_tokens = tokens if tokens >= 16 and rng.random() < 0.6 else _log_int(rng, 16, 9216)
        lengths = batch > 1 and rng.random() < 0.5
        while kv_heads > 1 and batch * kv_heads * group * tokens * kv_tokens * dim > 3.4e11:
            kv_heads -= 1
        if batch * kv_heads * group * tokens * kv_tokens * dim > 3.4e11:
            group = 1
        return _train(dtype, batch, kv_heads * group, kv_heads, tokens, kv_tokens, dim, lengths)
    dtype = rng.choice((dtype, dtype, "fp32"))
    dim = rng.choice((64, 80, 128, 128, 8 * rng.randint(2, 32)))
    rotated = dim if rng.random() < 0.6 else 8 * rng.randint(1, dim // 8)
    positions = rng.choice(("grid", "int", "float"))
    axes = _split_axes(rng, rotated, 3 if positions == "grid" else rng.randint(1, 3))
    batch, heads = rng.randint(1, 4), rng.randint(1, 40)
    grid = {}
    if positions == "grid":
        grid = {"frames": rng.randint(1, 16), "height": rng.randint(1, 64), "width": rng.randint(1, 64)}
        tokens = math.prod(grid.values())
    else:
        tokens = _log_int(rng, 1, 32768)
    heads = max(1, min(heads, int(40 * 32768 * 128 / (2 * batch * tokens * dim * (2 if dtype == "fp32" else 1)))))
    pairs = rng.random() < 0.5
    if kind == "rope":
        return _rope(dtype, batch, heads, tokens, dim, axes, positions, pairs, **grid)
    k_heads = max(1, heads // rng.choice((1, 1, 2, 4)))
    fused = k_heads == heads and rng.random() < 0.3
    return _norm(dtype, batch, heads, k_heads, tokens, dim, axes, positions, pairs, rng.random() < 0.5, fused, **grid)


# ------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * spread).to(dtype)


def _heads_first(x):
    """[B,T,H,D] storage as the [B,H,T,D] view that the attention calls take."""
    return x.permute(0, 2, 1, 3)


def _frequencies(axes):
    return torch.cat([_THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d) for d in axes])


def _positions(case, gen, axes):
    b, t = case["batch"], case["tokens"]
    if case["positions"] == "grid":
        return None
    if case["positions"] == "int":  # each sequence goes on from where it stands
        start = torch.randint(0, 100000, (b, 1, len(axes)), generator=gen, device="cuda")
        return start + torch.arange(t, device="cuda")[None, :, None]
    return torch.rand((t, len(axes)), generator=gen, device="cuda") * 128.0  # seconds, rows and columns


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, t, d = _DTYPES[case["dtype"]], case["batch"], case["tokens"], case["dim"]
    state = dict(case)
    if case["kind"] == "train":
        h, hk, tk = case["heads"], case["kv_heads"], case["kv_tokens"]
        # queries and keys as a norm with learned weights leaves them
        state["q"] = _heads_first(_normal(gen, (b, t, h, d), dtype, 1.2))
        state["k"] = _heads_first(_normal(gen, (b, tk, hk, d), dtype, 1.2))
        state["v"] = _heads_first(_normal(gen, (b, tk, hk, d), dtype))
        state["grad"] = _heads_first(_normal(gen, (b, t, h, d), dtype, 0.1))
        state["scale"] = d ** -0.5
        state["kv_lengths"] = None
        if case["lengths"]:
            lengths = torch.randint(tk // 8, tk + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
            lengths[0] = tk
            if b > 2:
                lengths[b - 1] = 0  # no text at all
            state["kv_lengths"] = lengths
        return state
    axes = state["axes"] = tuple(int(x) for x in case["axes"].split(","))
    state["inv_freq"] = _frequencies(axes)
    state["pos"] = _positions(case, gen, axes)
    state["grid"] = (case["frames"], case["height"], case["width"]) if case["positions"] == "grid" else None
    h = case["heads"]
    if case["kind"] == "rope":
        state["x"] = _heads_first(_normal(gen, (b, t, h, d), dtype))
        return state
    hk = case["k_heads"]
    if case["fused_qkv"]:
        qkv = _normal(gen, (b, t, 3, h, d), dtype, 2.0)
        state["q"], state["k"] = _heads_first(qkv[:, :, 0]), _heads_first(qkv[:, :, 1])
    else:
        state["q"] = _heads_first(_normal(gen, (b, t, h, d), dtype, 2.0))
        state["k"] = _heads_first(_normal(gen, (b, t, hk, d), dtype, 0.5))
    state["qw"] = (1.0 + _normal(gen, (d,), torch.float32, 0.2)).to(dtype)
    state["kw"] = (1.0 + _normal(gen, (d,), torch.float32, 0.2)).to(dtype)
    if case["grad"]:
        state["gq"] = _heads_first(_normal(gen, (b, t, h, d), dtype, 0.1))
        state["gk"] = _heads_first(_normal(gen, (b, t, hk, d), dtype, 0.1))
    return state


# ------------------------------------------------------------------ the plain forms
def _token_positions(s):
    """[1 or B, T, A] positions in 64 bits."""
    if s["grid"] is None:
        return s["pos"].double().reshape(-1, s["tokens"], len(s["axes"]))
    f, h, w = s["grid"]
    t = torch.arange(f * h * w, device="cuda")
    return torch.stack((t // (h * w), t // w % h, t % w), dim=-1).double()[None]


def _cos_sin(s):
    """[1 or B, 1, T, R/2] each; the angles in 64 bits (a far position times a frequency loses its turn in 32)."""
    axis = torch.repeat_interleave(torch.arange(len(s["axes"]), device="cuda"),
                                   torch.tensor([d // 2 for d in s["axes"]], device="cuda"), output_size=sum(s["axes"]) // 2)
    angle = _token_positions(s)[:, :, axis] * s["inv_freq"]
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(x, cos, sin, interleaved):
    """The first R dims of fp32 x rotated by pairs."""
    half = cos.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_norm(x, w, cos, sin, interleaved):
    xf = x.float()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + _EPS)
    return _rotate(xf * r * w.float(), cos, sin, interleaved).to(x.dtype)


def _plain_norm_backward(g, x, w, cos, sin, interleaved):
    xf = x.float()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + _EPS)
    n = xf * r
    g = _rotate(g.float(), cos, -sin, interleaved)
    dw = (g * n).double().sum((0, 1, 2)).to(w.dtype)
    a = g * w.float()
    return (r * (a - n * (a * n).mean(-1, keepdim=True))).to(x.dtype), dw


def _plain_train(s):
    q, k, v, g = (s[n].float().contiguous() for n in ("q", "k", "v", "grad"))
    (b, h, t, d), hk, tk = q.shape, k.shape[1], k.shape[2]
    q, g = q.view(b, hk, -1, d), g.view(b, hk, -1, d)  # the rows of a group's heads one after the other
    scores = q.mul(s["scale"]) @ k.transpose(2, 3)
    if s["kv_lengths"] is not None:
        closed = torch.arange(tk, device="cuda") >= s["kv_lengths"][:, None, None, None]
        scores = scores.masked_fill_(closed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = top + total.log()
    p = p.div_(total.masked_fill(total == 0.0, 1.0))
    out = p @ v
    dv = p.transpose(2, 3) @ g
    ds = g @ v.transpose(2, 3)
    ds = ds.sub_((g * out).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ k).mul_(s["scale"])
    dk = (ds.transpose(2, 3) @ q).mul_(s["scale"])
    rows = (b, h, t, d)
    dtype = s["q"].dtype
    return [out.view(rows).to(dtype), lse.view(b, h, t), dq.view(rows).to(dtype), dk.to(dtype), dv.to(dtype)]


# ------------------------------------------------------------------ one pass
def _package():
    if "mi355x_pisa" not in sys.modules:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "comfyui-rdna35-attention_amd"))
    import mi355x_pisa

    return mi355x_pisa


def _own_run(s):
    ops = _package()
    if s["kind"] == "train":
        out, lse = ops.dense_attention_with_lse(s["q"], s["k"], s["v"], s["scale"], kv_lengths=s["kv_lengths"])
        return [out, lse, *ops.dense_attention_backward(s["grad"], s["q"], s["k"], s["v"], out, lse, s["scale"],
                                                        kv_lengths=s["kv_lengths"])]
    turn = {"inv_freq": s["inv_freq"], "axes_dims": s["axes"], "positions": s["pos"], "token_grid": s["grid"],
            "interleaved": s["interleaved"]}
    if s["kind"] == "rope":
        return [ops.axial_rope(s["x"], **turn)]
    outs = list(ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], eps=_EPS, **turn))
    if s["grad"]:
        outs += ops.qk_norm_rope_backward(s["gq"], s["gk"], s["q"], s["k"], s["qw"], s["kw"], eps=_EPS, **turn)
    return outs


def run(state):
    s = state
    if own:
        return _own_run(s)
    if s["kind"] == "train":
        return _plain_train(s)
    cos, sin = _cos_sin(s)
    pairs = s["interleaved"]
    if s["kind"] == "rope":
        return [_rotate(s["x"].float(), cos, sin, pairs).to(s["x"].dtype)]
    outs = [_plain_norm(s["q"], s["qw"], cos, sin, pairs), _plain_norm(s["k"], s["kw"], cos, sin, pairs)]
    if s["grad"]:
        dq, dqw = _plain_norm_backward(s["gq"], s["q"], s["qw"], cos, sin, pairs)
        dk, dkw = _plain_norm_backward(s["gk"], s["k"], s["kw"], cos, sin, pairs)
        outs += [dq, dk, dqw, dkw]
    return outs


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    b, t, d = case["batch"], case["tokens"], case["dim"]
    if case["kind"] == "train":
        rows, keys = b * case["heads"] * t * d, b * case["kv_heads"] * case["kv_tokens"] * d
        # where there are lengths, they lie between an eighth and all of the keys (the first: all, a third: none)
        share = 1.0 if not case["lengths"] else (1.0 + 9 / 16 * (1 if b > 1 else 0)) / b
        return {"bytes": es * (4 * rows + 4 * keys) + 4 * rows // d, "flops": 14.0 * rows * case["kv_tokens"] * share}
    heads = case["heads"] + case.get("k_heads", 0)
    values = b * t * heads * d
    passes = 5 if case.get("grad") else 2
    return {"bytes": es * passes * values, "flops": values * {"rope": 3, "norm": 25 if case.get("grad") else 7}[case["kind"]]}


# ------------------------------------------------------------------ in 64 bits, from the definition
def _turned(x, s):
    """x's pairs as complex numbers times exp(i angle)."""
    parts, first = [], 0
    where = _token_positions(s)
    for axis, dims in enumerate(s["axes"]):
        angle = where[:, None, :, axis, None] * s["inv_freq"][first:first + dims // 2]
        parts.append(torch.polar(torch.ones_like(angle), angle))
        first += dims // 2
    unit, rotated = torch.cat(parts, dim=-1), 2 * first
    y = x.clone()
    if s["interleaved"]:
        z = torch.complex(x[..., 0:rotated:2], x[..., 1:rotated:2]) * unit
        y[..., 0:rotated:2], y[..., 1:rotated:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :first], x[..., first:rotated]) * unit
        y[..., :first], y[..., first:rotated] = z.real, z.imag
    return y


def _exact_norm(x, w, s):
    return _turned(x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w, s)


def _exact_train(s):
    """Head by head; the gradients are those of the forward's definition."""
    b, h, t, d = s["q"].shape
    hk, tk = s["k"].shape[1], s["k"].shape[2]
    out = torch.zeros((b, h, t, d), dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, t), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk = torch.zeros_like(out), torch.zeros((b, hk, tk, d), dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    counts = [tk] * b if s["kv_lengths"] is None else s["kv_lengths"].tolist()
    for i, n in enumerate(counts):
        for j in range(h if n else 0):
            c = j // (h // hk)
            q, k, v = (x.double().clone().requires_grad_() for x in (s["q"][i, j], s["k"][i, c, :n], s["v"][i, c, :n]))
            z = s["scale"] * torch.matmul(q, k.t())
            logs = torch.logsumexp(z, dim=1)
            o = torch.matmul(torch.exp(z - logs[:, None]), v)
            gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["grad"][i, j].double())
            out[i, j], lse[i, j], dq[i, j] = o.detach(), logs.detach(), gq
            dk[i, c, :n] += gk
            dv[i, c, :n] += gv
            del z, logs, o
    return [out, lse, dq, dk, dv]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "train":
        return _exact_train(s)
    if case["kind"] == "rope":
        return [_turned(s["x"].double(), s)]
    outs, grads, weights = [], [], []
    for x, w, g in (("q", "qw", "gq"), ("k", "kw", "gk")):
        leaf = [s[n].double().clone().requires_grad_(case["grad"]) for n in (x, w)]
        y = _exact_norm(*leaf, s)
        outs.append(y.detach())
        if case["grad"]:
            dx, dw = torch.autograd.grad(y, leaf, s[g].double())
            grads.append(dx)
            weights.append(dw)
        del y
    return outs + grads + weights
