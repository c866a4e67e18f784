"""64-bit references of the norm and the rotation, with the size of the fp32 error their kernels may make."""
from __future__ import annotations

import torch

STEP = 2.0 ** -24  # half a step of fp32, relative


def rounding(t: torch.dtype, value: torch.Tensor) -> torch.Tensor:
    """The most that rounding `value` to t moves it (subnormal steps included)."""
    info = torch.finfo(t)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def grid_positions(frames: int, height: int, width: int) -> torch.Tensor:
    f, y, x = torch.meshgrid(torch.arange(frames), torch.arange(height), torch.arange(width), indexing="ij")
    return torch.stack((f.flatten(), y.flatten(), x.flatten()), dim=-1)


def angles(inv_freq: torch.Tensor, axes, positions: torch.Tensor) -> torch.Tensor:
    """[1 or B, 1, T, R/2] in 64 bits."""
    pos = positions.double().cpu()
    pos = pos[None] if pos.ndim == 2 else pos
    parts, at = [], 0
    for i, d in enumerate(axes):
        parts.append(pos[:, :, i, None] * inv_freq.cpu()[at:at + d // 2])
        at += d // 2
    return torch.cat(parts, dim=-1)[:, None]


def pairs(x: torch.Tensor, rotated: int, interleaved: bool):
    if interleaved:
        return x[..., 0:rotated:2], x[..., 1:rotated:2]
    return x[..., :rotated // 2], x[..., rotated // 2:rotated]


def join(a: torch.Tensor, b: torch.Tensor, rest: torch.Tensor, interleaved: bool) -> torch.Tensor:
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def rotate(x: torch.Tensor, angle: torch.Tensor | None, interleaved: bool):
    """(rotated x, sum of the magnitudes that each of its dims is made of), x in 64 bits on the CPU.

    The magnitudes grow by 2^-30 of the angle: position * inv_freq is rounded to
    64 bits here, and in the kernel that product, 1 / (2 pi) and the product of
    the two are, so the angles differ by at most 4 * 2^-53 of their size, which
    is 8 steps of fp32 times 2^-30 (a position of 2^40 leaves 1e-3 of a radian).
    """
    if angle is None:
        return x, x.abs()
    rotated = 2 * angle.shape[-1]
    a, b = pairs(x, rotated, interleaved)
    c, s = angle.cos(), angle.sin()
    size = (a.abs() + b.abs()) * (1 + angle.abs() * 2.0 ** -30)
    return (join(a * c - b * s, a * s + b * c, x[..., rotated:], interleaved),
            join(size, size, x[..., rotated:].abs(), interleaved))


def norm_rope(x, w, eps, angle, interleaved):
    """y and the fp32 error its kernel may make, before the output's rounding.

    The sum of squares adds at most 13 roundings in a row (8 in a lane, 5
    exchanges), which the root halves; mean, eps, root, quotient and the two
    products add 7; an angle's fraction of a turn is off by 2^-26, hence its
    cosine by 2 pi 2^-26 < 2 steps, and by 2 more in its evaluation; the
    rotation adds 3: below 20 steps in all.
    """
    x = x.double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y, size = rotate(n * w, angle, interleaved)
    return y, 20 * STEP * size


def norm_rope_grad(g, x, w, eps, angle, interleaved):
    """(dx, its fp32 error, dw, its fp32 error) from the formulas.

    dx: g's pairs, a = g w and n are off by at most 20 steps each as above, the
    mean of a n by 20 more, and the result takes 4: below 64 steps of the terms'
    magnitudes.  dw: each term is off by 40 steps, and the sum adds at most one
    a row and 40 for joining the parts.
    """
    g, x = g.double().cpu(), x.double().cpu()
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = x * r
    back, size = rotate(g, None if angle is None else -angle, interleaved)
    a = back * wd
    dx = r * (a - n * (a * n).mean(-1, keepdim=True))
    spread = size * wd.abs()
    dx_size = r * (spread + n.abs() * (spread * n.abs()).mean(-1, keepdim=True))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (back * n).sum((0, 1, 2))
    dw_size = (size * n.abs()).sum((0, 1, 2))
    return dx, 64 * STEP * dx_size, dw, (rows + 80) * STEP * dw_size
