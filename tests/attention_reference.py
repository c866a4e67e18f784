"""64-bit reference of exact attention and its gradients, with the size of the error the kernels may make.

u is half a step of the input type, relative (what rounding to it costs).  The
kernels form scores, sums and gradients in fp32 and round P and dS to the
input type for their second products; the bounds follow each of these.
"""
from __future__ import annotations

import math

import torch

STEP = 2.0 ** -24  # half a step of fp32, relative
# The exponential and the matrix core take what lies below the smallest normal
# fp32 (and bf16) number as zero.
FLUSH = 2.0 ** -126


def _per_query_head(x, heads):
    return x.repeat_interleave(heads // x.shape[1], dim=1)


def _per_kv_head(x, kv_heads):
    b, h, t, d = x.shape
    return x.view(b, kv_heads, h // kv_heads, t, d).sum(2)


def reference(q, k, v, scale, kv_lengths=None, grad_out=None, grad_lse=None):
    """{name: (value, error)} of out and lse, and of dq, dk, dv where grad_out is given."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    half = dtype == torch.float16
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    batch, heads, _, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    if kv_lengths is not None:
        counts = kv_lengths.cpu().clamp(0, keys)
        open_ = (torch.arange(keys)[None] < counts[:, None])[:, None, None]
        k = torch.where(open_[:, :, 0, :, None], k, 0.0)  # what stands in masked keys has no say
        v = torch.where(open_[:, :, 0, :, None], v, 0.0)
    else:
        open_ = torch.ones((batch, 1, 1, keys), dtype=torch.bool)
    kq, vq = _per_query_head(k, heads), _per_query_head(v, heads)
    s = scale * q @ kq.transpose(2, 3)
    s = s.masked_fill(~open_, -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    some = torch.isfinite(lse)
    p = torch.where(some[..., None], torch.exp(s - torch.where(some, lse, 0.0)[..., None]), 0.0)
    out = p @ vq
    # scores: a sum of D products, the scale and its fp32 rounding
    es = scale * (dim + 6) * STEP * (q.abs() @ kq.abs().transpose(2, 3))
    es_row = torch.where(open_, es, 0.0).amax(-1)
    # the exponent's fma rounds a number of the scores' size in log2 units, the exponential adds 2 steps
    size = torch.where(open_, s.abs(), 0.0).amax(-1)
    e_lse = es_row + STEP * (keys + 16 + 4 * size) + 4 * STEP * torch.where(some, lse, 0.0).abs()
    rel = 2 * (es_row + 4 * STEP * (size + 2))[..., None]
    pv = p @ vq.abs()
    # P rounded (fp16: at most 2^-25 more for each key where it is subnormal; the row's largest is at least 1)
    e_out = (u + rel + (keys + 16) * STEP) * pv + u * out.abs() + torch.finfo(dtype).tiny * u
    e_out = e_out + FLUSH * torch.where(open_, 1.0, 0.0).double() @ vq.abs()
    if half:
        e_out = e_out + 2.0 ** -25 * torch.where(open_, 1.0, 0.0).double() @ vq.abs()
    found = {"out": (out, e_out), "lse": (lse, torch.where(some, e_lse, 0.0))}
    if grad_out is None:
        return found
    g = grad_out.detach().double().cpu()
    dl = torch.zeros_like(lse) if grad_lse is None else grad_lse.detach().double().cpu()
    rows = q.shape[2]
    dp = g @ vq.transpose(2, 3)
    delta = (g * out).sum(-1)
    diff = torch.where(open_, dp - delta[..., None] + dl[..., None], 0.0)
    ds = p * diff
    # P from the log sums: the scores' and the log sum's errors, the rounding of both in log2 units, the exponential
    r = (es_row + e_lse + 4 * STEP * (size + torch.where(some, lse, 0.0).abs() + 2))[..., None]
    e_delta = (g.abs() * e_out).sum(-1) + (dim + 8) * STEP * (g.abs() * out.abs()).sum(-1) + 2 * STEP * dl.abs()
    e_dp = (dim + 8) * STEP * (g.abs() @ vq.abs().transpose(2, 3) + delta.abs()[..., None] + dl.abs()[..., None])
    e_ds = p * (e_delta[..., None] + e_dp) * (1 + r) + (r + u + 4 * STEP) * (ds.abs() + p * (e_delta[..., None] + e_dp))
    e_p = (r + u) * p + torch.where(open_, FLUSH, 0.0)
    e_ds = e_ds + torch.where(open_, FLUSH, 0.0) * (1 + diff.abs())
    if half:
        # P times 2^15 and dS times 2^e: subnormal steps of 2^-25, scaled back; 2^-e is below the bound on
        # |diff| times 2^-14
        most = 2 * g.norm(dim=-1).amax(-1) * vq.norm(dim=-1).amax(-1) + dl.abs().amax(-1)
        most = _per_query_head(most.view(batch, kv_heads, -1).amax(-1, keepdim=True), heads)  # over a group's heads
        e_p = e_p + 2.0 ** -40 * (p > 0)
        e_ds = e_ds + 2.0 ** -39 * most[..., None] * (p > 0)
    pt, ept, dst, edst = (x.transpose(2, 3) for x in (p, e_p, ds, e_ds))
    tiny = torch.finfo(dtype).tiny * u

    def rounded(value, error, terms, count):
        error = error + (count + 16) * STEP * (terms + error)
        return value, error + u * (value.abs() + error) + tiny

    group = heads // kv_heads
    found["dq"] = rounded(scale * ds @ kq, scale * e_ds @ kq.abs(), scale * ds.abs() @ kq.abs(), keys)
    found["dk"] = rounded(_per_kv_head(scale * dst @ q, kv_heads), _per_kv_head(scale * edst @ q.abs(), kv_heads),
                          _per_kv_head(scale * dst.abs() @ q.abs(), kv_heads), rows * group)
    found["dv"] = rounded(_per_kv_head(pt @ g, kv_heads), _per_kv_head(ept @ g.abs(), kv_heads),
                          _per_kv_head(pt @ g.abs(), kv_heads), rows * group)
    return found


def near(actual, want, what):
    value, error = want
    a = actual.detach().double().cpu()
    assert a.shape == value.shape, (what, a.shape, value.shape)
    same = (a == value) | ((a - value).abs() <= error * (1 + 2.0 ** -6))
    if not bool(same.all()):
        worst = ((a - value).abs() / error.clamp_min(1e-300))[~same]
        raise AssertionError(f"{what}: {int((~same).sum())} of {a.numel()} off, worst {float(worst.max()):.3g} of the bound, "
                             f"first at {torch.nonzero(~same)[:3].tolist()}")
