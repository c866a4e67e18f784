"""Norm of queries and keys for each head and their rotation by position.

What a diffusion transformer does between its QKV projection and its
attention: an RMS norm of every head's row with a learned weight, then the
rotation of the row's pairs by the token's position along one to four axes
(time, height, width, ...).  The kernels (csrc/qk_norm_rope.hip) read each row
once and write it once; ``qk_norm_rope`` does both steps in one launch,
``axial_rope`` the rotation alone.  Both are differentiable;
``qk_norm_rope_backward`` is the backward pass as a plain call.

The models of the reference do these steps in torch before they call its
attention override; it has no kernel of this kind.
"""
from __future__ import annotations

import math
from collections.abc import Sequence
from typing import Optional

import torch

from . import _eager, _is_rocm_device, _lib
from ._lib import LIB, check, dtype_code, on_device, ptr, stream_of, view4

ROPE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
ROPE_HEAD_DIMS = tuple(range(8, 257, 8))
ROPE_MAX_AXES = 4
_POSITION_KINDS = {torch.int32: _lib.POSITIONS_I32, torch.int64: _lib.POSITIONS_I64, torch.float32: _lib.POSITIONS_F32}
_NO_VIEW = _lib.PisaView(None, 0, 0, 0)


def rope_frequencies(axes_dims: Sequence[int], theta: float | Sequence[float] = 10000.0, device=None) -> torch.Tensor:
    """float64 [sum(axes_dims)/2]: theta**(-2i/d) for pair i of each axis of d dims; theta may differ per axis."""
    dims = [int(d) for d in axes_dims]
    if not dims or any(d <= 0 or d % 2 for d in dims):
        raise ValueError("axes_dims must be positive even numbers")
    thetas = [float(x) for x in theta] if isinstance(theta, Sequence) else [float(theta)] * len(dims)
    if len(thetas) != len(dims) or not all(math.isfinite(x) and x > 0 for x in thetas):
        raise ValueError("theta must be positive and finite, one number or one for each axis")
    parts = [x ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d, x in zip(dims, thetas)]
    return torch.cat(parts).to(device) if device is not None else torch.cat(parts)


# --------------------------------------------------------------------------- checks
def _check_rows(what: str, name: str, x, like=None) -> None:
    """Every attribute is read once: these checks bound small calls."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor.")
    shape = x.shape
    if len(shape) != 4 or 0 in shape:
        raise ValueError(f"{what}: {name} must be [B,H,T,D] with every dimension positive, got {tuple(shape)}")
    if not _is_rocm_device(x):
        raise ValueError(f"{what}: {name} must be on a PyTorch ROCm device.")
    if x.dtype not in ROPE_DTYPES:
        raise ValueError(f"{what}: {name} must be bfloat16, float16 or float32, got {x.dtype}")
    if shape[3] % 8 or shape[3] > 256:
        raise ValueError(f"{what}: head dim must be a multiple of 8 up to 256, got {shape[3]}")
    if x.stride(3) != 1:
        raise ValueError(f"{what}: {name}'s head_dim must have unit stride")
    if like is not None:
        other = like.shape
        if shape[0] != other[0] or shape[2] != other[2] or shape[3] != other[3]:
            raise ValueError(f"{what}: {name} {tuple(shape)} must share batch, tokens and head dim with {tuple(other)}")
        if x.device != like.device or x.dtype != like.dtype:
            raise ValueError(f"{what}: {name} must share q's device and dtype")


def _check_weights(what: str, q, weights) -> None:
    first = None
    for w in weights:
        if w is None:
            continue
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{what}: weights must be torch tensors.")
        if w.ndim != 1 or w.shape[0] != q.shape[3] or w.device != q.device or not w.is_contiguous():
            raise ValueError(f"{what}: a weight must be contiguous [{q.shape[3]}] on q's device, got {tuple(w.shape)}")
        first = w.dtype if first is None else first
        if w.dtype != first or (first != torch.float32 and first != q.dtype):
            raise ValueError(f"{what}: weights must share one dtype, q's or float32, got {w.dtype}")


def _check_eps(what: str, eps) -> float:
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"{what}: eps must be finite and not negative")
    return eps


def _check_rotation(what: str, x, inv_freq, axes_dims, positions, token_grid) -> tuple[int, ...]:
    """The axes' dims () without a rotation."""
    if inv_freq is None:
        if axes_dims is not None or positions is not None or token_grid is not None:
            raise ValueError(f"{what}: axes_dims, positions and token_grid need inv_freq")
        return ()
    if axes_dims is None or not 1 <= len(axes_dims) <= ROPE_MAX_AXES:
        raise ValueError(f"{what}: axes_dims must name 1 to {ROPE_MAX_AXES} axes")
    axes = tuple([int(d) for d in axes_dims])
    rotated = sum(axes)
    if rotated % 8 or rotated > x.shape[3] or min(axes) <= 0 or any([d % 2 for d in axes]):
        raise ValueError(f"{what}: axes_dims {axes} must be positive even numbers whose sum is a multiple of 8 and at "
                         f"most the head dim {x.shape[3]}")
    if not isinstance(inv_freq, torch.Tensor):
        raise TypeError(f"{what}: inv_freq must be a torch tensor.")
    if inv_freq.dtype != torch.float64 or tuple(inv_freq.shape) != (rotated // 2,) or not inv_freq.is_contiguous() \
            or inv_freq.device != x.device:
        raise ValueError(f"{what}: inv_freq must be contiguous float64 [{rotated // 2}] on the input's device")
    if inv_freq.requires_grad:
        raise ValueError(f"{what}: inv_freq has no gradient here")
    if (positions is None) == (token_grid is None):
        raise ValueError(f"{what}: give either positions or token_grid")
    batch, tokens = x.shape[0], x.shape[2]
    if token_grid is not None:
        frames, height, width = (int(n) for n in token_grid)
        if len(axes) != 3 or min(frames, height, width) <= 0 or frames * height * width != tokens:
            raise ValueError(f"{what}: token_grid {tuple(token_grid)} needs 3 axes and {tokens} tokens")
        return axes
    if not isinstance(positions, torch.Tensor):
        raise TypeError(f"{what}: positions must be a torch tensor.")
    if positions.dtype not in _POSITION_KINDS or positions.device != x.device:
        raise ValueError(f"{what}: positions must be int32, int64 or float32 on the input's device")
    where = positions.shape
    if where[-2:] != (tokens, len(axes)) or len(where) not in (2, 3) or (len(where) == 3 and where[0] not in (1, batch)):
        raise ValueError(f"{what}: positions must be [T,A] or [B,T,A] with T={tokens} and A={len(axes)}, got "
                         f"{tuple(positions.shape)}")
    if positions.requires_grad:
        raise ValueError(f"{what}: positions have no gradient here")
    return axes


# --------------------------------------------------------------------------- launchers
_DIMS = _lib.ctypes.c_int32 * ROPE_MAX_AXES
_NO_GRID = _lib.grid()


def _rope_struct(inv_freq, axes, positions, grid, interleaved: bool, inverse: bool) -> _lib.PisaRope:
    if not axes:
        return _lib.PisaRope(None, None, 0, 0, 0, _NO_GRID, 0, 0, _DIMS(), interleaved, inverse)
    dims = _DIMS(*axes)
    if positions is None:
        return _lib.PisaRope(inv_freq.data_ptr(), None, 0, 0, 0, _lib.grid(*grid), _lib.POSITIONS_GRID, len(axes), dims,
                             interleaved, inverse)
    strides = positions.stride()
    batch = strides[0] if len(strides) == 3 and positions.shape[0] > 1 else 0
    return _lib.PisaRope(inv_freq.data_ptr(), positions.data_ptr(), batch, strides[-2], strides[-1], _NO_GRID,
                         _POSITION_KINDS[positions.dtype], len(axes), dims, interleaved, inverse)


def _heads_last(x) -> torch.Tensor:
    """An empty [B,H,T,D] view of contiguous [B,T,H,D] storage, the layout that the attention calls read best."""
    batch, heads, tokens, dim = x.shape
    return torch.empty_strided((batch, heads, tokens, dim), (tokens * heads * dim, dim, heads * dim, 1), dtype=x.dtype,
                               device=x.device)


def _view(x) -> _lib.PisaView:
    return _NO_VIEW if x is None else view4(x)


def _weight_code(q, *weights) -> int:
    return next((dtype_code(w.dtype) for w in weights if w is not None), dtype_code(q.dtype))


def _forward_kernel(q, k, q_weight, k_weight, eps: float, normalize: bool, inv_freq, axes, positions, grid,
                    interleaved: bool, inverse: bool):
    batch, heads, tokens, dim = q.shape
    q_out, k_out = _heads_last(q), None if k is None else _heads_last(k)
    with on_device(q.device):
        check(
            LIB.attn_hip_qk_norm_rope(
                dtype_code(q.dtype), _weight_code(q, q_weight, k_weight), batch, heads,
                0 if k is None else k.shape[1], tokens, dim, view4(q), _view(k), view4(q_out), _view(k_out),
                ptr(q_weight), ptr(k_weight), int(normalize), eps,
                _rope_struct(inv_freq, axes, positions, grid, interleaved, inverse), stream_of(q.device),
            ),
            "attn_hip_qk_norm_rope",
        )
    return q_out, k_out


def _backward_kernel(grad_q, grad_k, q, k, q_weight, k_weight, eps: float, inv_freq, axes, positions, grid,
                     interleaved: bool):
    batch, heads, tokens, dim = q.shape
    dq, dk = _heads_last(q), None if k is None else _heads_last(k)
    dqw, dkw = (None if w is None else torch.empty_like(w) for w in (q_weight, k_weight))
    with on_device(q.device):
        ws_bytes = LIB.attn_hip_qk_norm_rope_backward_workspace_bytes(dim, int(dqw is not None or dkw is not None))
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        check(
            LIB.attn_hip_qk_norm_rope_backward(
                dtype_code(q.dtype), _weight_code(q, q_weight, k_weight), batch, heads,
                0 if k is None else k.shape[1], tokens, dim, view4(grad_q), _view(grad_k), view4(q), _view(k),
                ptr(q_weight), ptr(k_weight), view4(dq), _view(dk), ptr(dqw), ptr(dkw), eps,
                _rope_struct(inv_freq, axes, positions, grid, interleaved, False), ptr(workspace), ws_bytes,
                stream_of(q.device),
            ),
            "attn_hip_qk_norm_rope_backward",
        )
    return dq, dk, dqw, dkw


def _unit_stride(grad, like):
    """An incoming gradient with unit head_dim stride (autograd may hand on an expanded one)."""
    if grad is None:
        return torch.zeros_like(like)
    return grad if grad.stride(3) == 1 else grad.contiguous()


# --------------------------------------------------------------------------- custom ops
# Registered like the package's other ops, with fake implementations and, since
# these are differentiable, autograd formulas: both trace under torch.compile.
# Eager calls run the kernels through torch.autograd.Function (or directly
# when nothing requires a gradient), without the dispatcher.
def _fake_rows(x):
    return x.new_empty((x.shape[0], x.shape[2], x.shape[1], x.shape[3])).permute(0, 2, 1, 3)


@torch.library.custom_op("mi355x_pisa::axial_rope", mutates_args=(), device_types="cuda")
def _axial_rope_op(x: torch.Tensor, inv_freq: torch.Tensor, axes: Sequence[int], positions: Optional[torch.Tensor],
                   grid: Sequence[int], interleaved: bool, inverse: bool) -> torch.Tensor:
    return _forward_kernel(x, None, None, None, 0.0, False, inv_freq, tuple(axes), positions, tuple(grid), interleaved,
                           inverse)[0]


@_axial_rope_op.register_fake
def _axial_rope_op_fake(x, inv_freq, axes, positions, grid, interleaved, inverse):
    del inv_freq, axes, positions, grid, interleaved, inverse
    return _fake_rows(x)


def _axial_rope_setup(ctx, inputs, output):
    x, inv_freq, axes, positions, grid, interleaved, inverse = inputs
    del x, output
    ctx.save_for_backward(inv_freq, positions)
    ctx.args = (axes, grid, interleaved, inverse)


def _axial_rope_grad(ctx, grad):
    inv_freq, positions = ctx.saved_tensors
    axes, grid, interleaved, inverse = ctx.args
    dx = _axial_rope_op(_unit_stride(grad, grad), inv_freq, axes, positions, grid, interleaved, not inverse)
    return dx, None, None, None, None, None, None


_axial_rope_op.register_autograd(_axial_rope_grad, setup_context=_axial_rope_setup)


@torch.library.custom_op("mi355x_pisa::qk_norm_rope", mutates_args=(), device_types="cuda")
def _qk_norm_rope_op(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                     k_weight: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor],
                     axes: Sequence[int], positions: Optional[torch.Tensor], grid: Sequence[int],
                     interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    q_out, k_out = _forward_kernel(q, k, q_weight, k_weight, eps, True, inv_freq, tuple(axes), positions, tuple(grid),
                                   interleaved, False)
    return q_out, q.new_empty(0) if k_out is None else k_out


@_qk_norm_rope_op.register_fake
def _qk_norm_rope_op_fake(q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid, interleaved):
    del q_weight, k_weight, eps, inv_freq, axes, positions, grid, interleaved
    return _fake_rows(q), q.new_empty(0) if k is None else _fake_rows(k)


@torch.library.custom_op("mi355x_pisa::qk_norm_rope_backward", mutates_args=(), device_types="cuda")
def _qk_norm_rope_backward_op(grad_q: torch.Tensor, grad_k: Optional[torch.Tensor], q: torch.Tensor,
                              k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                              k_weight: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor],
                              axes: Sequence[int], positions: Optional[torch.Tensor], grid: Sequence[int],
                              interleaved: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    grads = _backward_kernel(grad_q, grad_k, q, k, q_weight, k_weight, eps, inv_freq, tuple(axes), positions,
                             tuple(grid), interleaved)
    return tuple(q.new_empty(0) if g is None else g for g in grads)


@_qk_norm_rope_backward_op.register_fake
def _qk_norm_rope_backward_op_fake(grad_q, grad_k, q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid,
                                   interleaved):
    del grad_q, grad_k, eps, inv_freq, axes, positions, grid, interleaved
    return (_fake_rows(q), q.new_empty(0) if k is None else _fake_rows(k),
            *(q.new_empty(0) if w is None else torch.empty_like(w) for w in (q_weight, k_weight)))


def _qk_norm_rope_setup(ctx, inputs, output):
    del output
    q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid, interleaved = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions)
    ctx.args = (eps, axes, grid, interleaved)


def _qk_norm_rope_grad(ctx, grad_q, grad_k):
    q, k, q_weight, k_weight, inv_freq, positions = ctx.saved_tensors
    eps, axes, grid, interleaved = ctx.args
    grads = _qk_norm_rope_backward_op(
        _unit_stride(grad_q, q), None if k is None else _unit_stride(grad_k, k), q, k, q_weight, k_weight, eps,
        inv_freq, axes, positions, grid, interleaved)
    inputs = (q, k, q_weight, k_weight)
    return (*(None if x is None else g for x, g in zip(inputs, grads)), None, None, None, None, None, None)


_qk_norm_rope_op.register_autograd(_qk_norm_rope_grad, setup_context=_qk_norm_rope_setup)


class _AxialRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, inv_freq, axes, positions, grid, interleaved, inverse):
        ctx.save_for_backward(inv_freq, positions)
        ctx.args = (axes, grid, interleaved, inverse)
        return _forward_kernel(x, None, None, None, 0.0, False, inv_freq, axes, positions, grid, interleaved, inverse)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        inv_freq, positions = ctx.saved_tensors
        axes, grid, interleaved, inverse = ctx.args
        dx = _forward_kernel(_unit_stride(grad, grad), None, None, None, 0.0, False, inv_freq, axes, positions, grid,
                             interleaved, not inverse)[0]
        return dx, None, None, None, None, None, None


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions)
        ctx.args = (eps, axes, grid, interleaved)
        return _forward_kernel(q, k, q_weight, k_weight, eps, True, inv_freq, axes, positions, grid, interleaved, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, inv_freq, positions = ctx.saved_tensors
        eps, axes, grid, interleaved = ctx.args
        grads = _backward_kernel(_unit_stride(grad_q, q), None if k is None else _unit_stride(grad_k, k), q, k,
                                 q_weight, k_weight, eps, inv_freq, axes, positions, grid, interleaved)
        return (*grads, None, None, None, None, None, None)


def _plain(*tensors) -> bool:
    """Eager call on plain tensors and parameters."""
    return _eager(*(t for t in tensors if type(t) is not torch.nn.Parameter))


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --------------------------------------------------------------------------- public API
def axial_rope(x: torch.Tensor, inv_freq: torch.Tensor, axes_dims: Sequence[int],
               positions: torch.Tensor | None = None, token_grid: tuple[int, int, int] | None = None,
               interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """x [B,H,T,D] with its pairs turned by position; returns a [B,H,T,D] view of [B,T,H,D] storage.

    Pair p of the first R = sum(axes_dims) dims is turned by the angle
    position[axis(p)] * inv_freq[p]: the first axes_dims[0]/2 pairs follow
    axis 0, the next axis 1, and so on.  Pair p is dims (2p, 2p+1) when
    `interleaved`, else (p, p + R/2); dims from R on pass unchanged.

    inv_freq    float64 [R/2] on x's device (rope_frequencies)
    axes_dims   1 to 4 even numbers, their sum a multiple of 8
    positions   int32/int64/float32 [T,A] or [B,T,A]; or
    token_grid  (frames, height, width): the tokens in raster order, 3 axes
    inverse     turn back

    x is bf16, fp16 or fp32, D a multiple of 8 up to 256, any strides with
    unit D stride.  Angles are formed in fp64, products in fp32.  Differentiable
    in x (once).
    """
    _check_rows("axial_rope", "x", x)
    if inv_freq is None:
        raise ValueError("axial_rope: inv_freq is needed")
    axes = _check_rotation("axial_rope", x, inv_freq, axes_dims, positions, token_grid)
    grid = (0, 0, 0) if token_grid is None else tuple(int(n) for n in token_grid)
    args = (x, inv_freq, axes, positions, grid, bool(interleaved), bool(inverse))
    if not _plain(x, inv_freq, positions):
        return _axial_rope_op(x, inv_freq, list(axes), positions, list(grid), *args[5:])
    if _wants_grad(x):
        return _AxialRope.apply(*args)
    return _forward_kernel(x, None, None, None, 0.0, False, *args[1:])[0]


def _check_norm_call(what, q, k, q_weight, k_weight, eps, inv_freq, axes_dims, positions, token_grid):
    _check_rows(what, "q", q)
    if k is not None:
        _check_rows(what, "k", k, like=q)
    elif k_weight is not None:
        raise ValueError(f"{what}: k_weight needs k")
    _check_weights(what, q, (q_weight, k_weight))
    axes = _check_rotation(what, q, inv_freq, axes_dims, positions, token_grid)
    return _check_eps(what, eps), axes, (0, 0, 0) if token_grid is None else tuple(int(n) for n in token_grid)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, *, eps: float = 1e-6, inv_freq: torch.Tensor | None = None,
                 axes_dims: Sequence[int] | None = None, positions: torch.Tensor | None = None,
                 token_grid: tuple[int, int, int] | None = None,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of every row of q [B,Hq,T,D] and k [B,Hk,T,D] and its rotation, in one pass.

    y = rotation(x * rsqrt(mean(x^2) + eps) * weight), one rounding at the end;
    the rotation's arguments are axial_rope's, none of them for the norm alone.
    Weights are [D] in q's dtype or float32 (None: ones).  k may be None
    (queries of a cross attention) and have another head count than q.
    Returns (q, k) as [B,H,T,D] views of [B,T,H,D] storage, which the attention
    calls take as they are.  Differentiable in q, k and the weights (once).
    """
    eps, axes, grid = _check_norm_call("qk_norm_rope", q, k, q_weight, k_weight, eps, inv_freq, axes_dims, positions,
                                       token_grid)
    args = (q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid, bool(interleaved))
    if not _plain(q, k, q_weight, k_weight, inv_freq, positions):
        q_out, k_out = _qk_norm_rope_op(*args[:6], list(axes), positions, list(grid), args[9])
        return q_out, None if k is None else k_out
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(*args)
    return _forward_kernel(q, k, q_weight, k_weight, eps, True, inv_freq, axes, positions, grid, bool(interleaved), False)


def qk_norm_rope_backward(grad_q: torch.Tensor, grad_k: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor | None,
                          q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, *,
                          eps: float = 1e-6, inv_freq: torch.Tensor | None = None,
                          axes_dims: Sequence[int] | None = None, positions: torch.Tensor | None = None,
                          token_grid: tuple[int, int, int] | None = None, interleaved: bool = False):
    """Gradients (dq, dk, dq_weight, dk_weight) of qk_norm_rope from those of its outputs.

    The other arguments are the forward call's; dk and the weights' gradients
    are None where there is no k or no such weight.  Sums over rows are fp32
    and taken in a fixed order, so the result is the same from run to run.
    """
    what = "qk_norm_rope_backward"
    eps, axes, grid = _check_norm_call(what, q, k, q_weight, k_weight, eps, inv_freq, axes_dims, positions, token_grid)
    if (grad_k is None) != (k is None):
        raise ValueError(f"{what}: grad_k and k go together")
    for name, g, x in (("grad_q", grad_q, q), ("grad_k", grad_k, k)):
        if x is not None:
            _check_rows(what, name, g, like=q)
            if g.shape != x.shape:
                raise ValueError(f"{what}: {name} must be {tuple(x.shape)}, got {tuple(g.shape)}")
    args = (grad_q, grad_k, q, k, q_weight, k_weight, eps, inv_freq, axes, positions, grid, bool(interleaved))
    if _plain(grad_q, grad_k, q, k, q_weight, k_weight, inv_freq, positions):
        return _backward_kernel(*args)
    grads = _qk_norm_rope_backward_op(*args[:8], list(axes), positions, list(grid), args[11])
    return tuple(None if x is None else g for x, g in zip((q, k, q_weight, k_weight), grads))
