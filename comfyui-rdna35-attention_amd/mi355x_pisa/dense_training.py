"""Exact attention for training: the forward with its rows' log sums, and the backward pass.

``dense_attention_with_lse`` is ``dense_attention`` with grouped key heads, a
key count per batch entry and a second output, the logarithm of every row's
sum of exponentials; it is differentiable.  ``dense_attention_backward`` is its
backward pass as a plain call: the probabilities are formed again from the log
sums (csrc/attention_backward.hip), so a layer keeps q, k, v, its output and
one number per row.

The reference is forward-only.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _HIP, _lib
from ._lib import LIB, check, dtype_code, on_device, ptr, stream_of, view4
from .rotary import _fake_rows, _heads_last, _plain, _wants_grad

TRAIN_DTYPES = (torch.bfloat16, torch.float16)
_NO_VIEW = _lib.PisaView(None, 0, 0, 0)


# --------------------------------------------------------------------------- checks
def _check_call(what: str, q, k, v, scale, kv_lengths) -> float:
    """Every attribute is read once: these checks bound small calls."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError(f"{what}: q, k, and v must be torch tensors.")
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise ValueError(f"{what}: expects [B,H,T,D] q/k/v, got {len(qs)}-D/{len(ks)}-D/{len(vs)}-D")
    if ks != vs:
        raise ValueError(f"{what}: k {tuple(ks)} and v {tuple(vs)} must match")
    if qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError(f"{what}: q {tuple(qs)} and k/v {tuple(ks)} must share batch and head dim")
    if 0 in qs or 0 in ks:
        raise ValueError(f"{what}: every dimension must be positive")
    if qs[1] % ks[1]:
        raise ValueError(f"{what}: {ks[1]} key heads do not divide {qs[1]} query heads")
    device, dtype = q.device, q.dtype
    if device != k.device or device != v.device or device.type != "cuda" or not _HIP:
        raise ValueError(f"{what}: q/k/v must be on one PyTorch ROCm device.")
    if dtype not in TRAIN_DTYPES or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{what}: q/k/v must share one dtype of bfloat16/float16, got {dtype}/{k.dtype}/{v.dtype}")
    if q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError(f"{what}: head_dim must have unit stride")
    if kv_lengths is not None:
        if not isinstance(kv_lengths, torch.Tensor):
            raise TypeError(f"{what}: kv_lengths must be a torch tensor.")
        if kv_lengths.dtype != torch.int32 or tuple(kv_lengths.shape) != (qs[0],) or kv_lengths.device != device \
                or not kv_lengths.is_contiguous():
            raise ValueError(f"{what}: kv_lengths must be contiguous int32 [{qs[0]}] on q's device")
    scale = float(scale)
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"{what}: scale must be positive and finite")
    return scale


# --------------------------------------------------------------------------- launchers
def _forward_kernel(q, k, v, scale: float, kv_lengths):
    batch, heads, q_tokens, head_dim = q.shape
    kv_heads, kv_tokens = k.shape[1], k.shape[2]
    out = _heads_last(q)
    lse = torch.empty((batch, heads, q_tokens), dtype=torch.float32, device=q.device)
    code = dtype_code(q.dtype)
    with on_device(q.device):
        ws_bytes = LIB.attn_hip_dense_forward_lse_workspace_bytes(code, batch, heads, kv_heads, q_tokens, kv_tokens, head_dim)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        check(
            LIB.attn_hip_dense_forward_lse(
                code, batch, heads, kv_heads, q_tokens, kv_tokens, head_dim, view4(q), view4(k), view4(v),
                view4(out), lse.data_ptr(), ptr(kv_lengths), scale, workspace.data_ptr(), ws_bytes, stream_of(q.device),
            ),
            "attn_hip_dense_forward_lse",
        )
    return out, lse


def _backward_kernel(grad_out, q, k, v, out, lse, scale: float, kv_lengths, grad_lse, need_q: bool = True,
                     need_kv: bool = True):
    batch, heads, q_tokens, head_dim = q.shape
    kv_heads, kv_tokens = k.shape[1], k.shape[2]
    dq = _heads_last(q) if need_q else None
    dk, dv = (_heads_last(k), _heads_last(v)) if need_kv else (None, None)
    code = dtype_code(q.dtype)
    with on_device(q.device):
        ws_bytes = LIB.attn_hip_dense_backward_workspace_bytes(code, batch, heads, kv_heads, q_tokens, kv_tokens, head_dim)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        check(
            LIB.attn_hip_dense_backward(
                code, batch, heads, kv_heads, q_tokens, kv_tokens, head_dim, view4(q), view4(k), view4(v), view4(out),
                view4(grad_out), lse.data_ptr(), ptr(grad_lse), ptr(kv_lengths), scale,
                *(_NO_VIEW if t is None else view4(t) for t in (dq, dk, dv)), workspace.data_ptr(), ws_bytes,
                stream_of(q.device),
            ),
            "attn_hip_dense_backward",
        )
    return dq, dk, dv


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """x if the kernels can read it (unit head_dim stride, 16-byte rows), else a copy: autograd hands on any layout."""
    s = x.stride()
    if s[3] == 1 and x.data_ptr() % 16 == 0 and not any(n % 8 for n in s[:3]):
        return x
    return x.clone(memory_format=torch.contiguous_format)


# --------------------------------------------------------------------------- custom ops
@torch.library.custom_op("mi355x_pisa::dense_attention_with_lse", mutates_args=(), device_types="cuda")
def _with_lse_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                 kv_lengths: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    return _forward_kernel(q, k, v, scale, kv_lengths)


@_with_lse_op.register_fake
def _with_lse_op_fake(q, k, v, scale, kv_lengths):
    del k, v, scale, kv_lengths
    return _fake_rows(q), q.new_empty(q.shape[:3], dtype=torch.float32)


@torch.library.custom_op("mi355x_pisa::dense_attention_backward", mutates_args=(), device_types="cuda")
def _backward_op(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                 lse: torch.Tensor, scale: float, kv_lengths: Optional[torch.Tensor],
                 grad_lse: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _backward_kernel(_rows16(grad_out), q, k, v, out, lse, scale, kv_lengths,
                            None if grad_lse is None else grad_lse.contiguous())


@_backward_op.register_fake
def _backward_op_fake(grad_out, q, k, v, out, lse, scale, kv_lengths, grad_lse):
    del grad_out, out, lse, scale, kv_lengths, grad_lse
    return _fake_rows(q), _fake_rows(k), _fake_rows(v)


def _with_lse_setup(ctx, inputs, output):
    q, k, v, scale, kv_lengths = inputs
    ctx.save_for_backward(q, k, v, kv_lengths, *output)
    ctx.scale = scale


def _with_lse_grad(ctx, grad_out, grad_lse):
    q, k, v, kv_lengths, out, lse = ctx.saved_tensors
    grad_out = torch.zeros_like(out) if grad_out is None else grad_out
    return (*_backward_op(grad_out, q, k, v, out, lse, ctx.scale, kv_lengths, grad_lse), None, None)


_with_lse_op.register_autograd(_with_lse_grad, setup_context=_with_lse_setup)


class _WithLse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, kv_lengths):
        ctx.set_materialize_grads(False)
        out, lse = _forward_kernel(q, k, v, scale, kv_lengths)
        ctx.save_for_backward(q, k, v, kv_lengths, out, lse)
        ctx.scale = scale
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_lse):
        q, k, v, kv_lengths, out, lse = ctx.saved_tensors
        grad_out = torch.zeros_like(out) if grad_out is None else _rows16(grad_out)
        grads = _backward_kernel(grad_out, q, k, v, out, lse, ctx.scale, kv_lengths,
                                 None if grad_lse is None else grad_lse.contiguous(), ctx.needs_input_grad[0],
                                 any(ctx.needs_input_grad[1:3]))
        return (*grads, None, None)


# --------------------------------------------------------------------------- public API
def dense_attention_with_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                             kv_lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Exact attention of [B,H,Tq,D] q over [B,Hkv,Tk,D] k/v, with the rows' log sums: (out, lse).

    bf16 or fp16, D a multiple of 8 up to 256; Hkv divides H (query heads
    h*H/Hkv .. share key head h); any strides with unit D stride and 16-byte
    rows.  kv_lengths (int32 [B] on q's device) masks the keys from
    kv_lengths[b] on; what stands in them is not used, and with no key left a
    row is 0 and its lse minus infinity.  out is a [B,H,Tq,D] view of
    [B,Tq,H,D] storage, lse fp32 [B,H,Tq] (natural logarithm).
    Differentiable in q, k and v through both outputs (once).
    """
    scale = _check_call("dense_attention_with_lse", q, k, v, scale, kv_lengths)
    if not _plain(q, k, v, kv_lengths):
        return _with_lse_op(q, k, v, scale, kv_lengths)
    if _wants_grad(q, k, v):
        return _WithLse.apply(q, k, v, scale, kv_lengths)
    return _forward_kernel(q, k, v, scale, kv_lengths)


def dense_attention_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             out: torch.Tensor, lse: torch.Tensor, scale: float,
                             kv_lengths: torch.Tensor | None = None,
                             grad_lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of dense_attention_with_lse from those of its outputs.

    out and lse are what the forward call returned for the same q, k, v, scale
    and kv_lengths; grad_lse (fp32 [B,H,Tq]) is the gradient of lse, None for
    zero.  dk and dv sum over the query heads of a group; masked keys get zero.
    The result is the same bit for bit from run to run.
    """
    what = "dense_attention_backward"
    scale = _check_call(what, q, k, v, scale, kv_lengths)
    for name, x in (("grad_out", grad_out), ("out", out)):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch tensor.")
        if x.shape != q.shape or x.dtype != q.dtype or x.device != q.device or x.stride(3) != 1:
            raise ValueError(f"{what}: {name} must be {tuple(q.shape)} of q's dtype and device with unit head_dim stride")
    for name, x in (("lse", lse), ("grad_lse", grad_lse)):
        if x is None and name == "grad_lse":
            continue
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch tensor.")
        if x.dtype != torch.float32 or x.shape != q.shape[:3] or x.device != q.device or not x.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous float32 {tuple(q.shape[:3])} on q's device")
    args = (grad_out, q, k, v, out, lse, scale, kv_lengths, grad_lse)
    if not _plain(*args[:6], kv_lengths, grad_lse):
        return _backward_op(*args)
    return _backward_kernel(*args)
