"""The learner's operators from their formulas, in float64 (torch on any
device): what the tests compare the kernels with, and the bounds on how far a
float32 evaluation rounded once to its type may be from them.
"""

from __future__ import annotations

import math

import torch

U32 = torch.finfo(torch.float32).eps / 2  # half a step of float32, relative


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to `dtype` (normal range)."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half the spacing of the subnormal numbers of `dtype`."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def layer_norm(x, w, b, eps):
    """y, mean, rstd of rows [R, D], in float64."""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    y = d * rstd
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def layer_norm_backward(dy, x, w, eps):
    """dx, dw, db of rows [R, D], in float64."""
    _, mean, rstd = layer_norm(x, None, None, eps)
    h = (x.double() - mean) * rstd
    dy = dy.double()
    g = dy if w is None else dy * w.double()
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def row_depth(dim: int) -> int:
    """Additions in float32 that a row's value passes through: up to 32 in one
    thread (longer rows join such sums in float64), the joins of a CTA or a
    cluster, and the handful of operations around them."""
    return 64


def row_error(x, rstd):
    """Rounding of a row's statistics, in units of its spread ([R, 1]).

    With n values, u = 2^-24 and a sum whose terms pass through at most m
    additions, |error of the sum| <= m u sum |terms|; e = m u below. Distances
    are taken from a first estimate s of the mean: of all values, off by at
    most e avg|x|, or of a quarter of a warp's values, off by at most sqrt(3)
    of its spread. The distances' mean square is then at most 4 / rstd^2 +
    (e avg|x|)^2, their sums pass through at most 32 additions (half of the 64
    in row_depth(), so that the factor 2 of their root mean square is counted),
    and the shift avg(x - s) is off by e (1 / rstd + e avg|x|), the variance,
    relative to var + eps, by 2 e (1 + (e avg|x| rstd)^2), which rstd halves."""
    e = row_depth(x.shape[1]) * U32
    far = e * x.double().abs().mean(1, keepdim=True) * rstd
    return e * (1 + far + far * far)


def layer_norm_bound(x, w, b, eps, dtype):
    """Bound on |y - layer_norm(...)| element by element: with E = row_error,
    h = (d - shift) rstd is off by at most (1 + |h|) E; multiplying by w and
    adding b adds u (|h w| + |y|), and the result is rounded once."""
    y, mean, rstd = layer_norm(x, w, b, eps)
    h = ((x.double() - mean) * rstd).abs()
    wa = 1.0 if w is None else w.double().abs()
    err = (1 + h) * wa * row_error(x, rstd) + 2 * U32 * y.abs()
    return y, err + half_step(dtype) * (y.abs() + err) + tiny(dtype)


def layer_norm_backward_bound(dy, x, w, eps, dtype, param_dtype):
    """The gradients and bounds on the distance from them.

    With e = row_error: h carries (1 + |h|) e, c1 = avg(g) e avg|g|,
    c2 = avg(g h) e avg(|g| (1 + 2 |h|)); dx = rstd (g - c1 - h c2) the sum of
    their shares plus the rounding of its own terms (each below e times its
    size). dw = sum dy h and db = sum dy pass through at most rows / 8 + 256
    additions (the partial sums and their join) on top of the error of h. Over
    many rows that bound exceeds the sums themselves; whole numbers that
    float32 adds exactly show a lost row there."""
    _, mean, rstd = layer_norm(x, None, None, eps)
    h = ((x.double() - mean) * rstd)
    dx, dw, db = layer_norm_backward(dy, x, w, eps)
    ha, dya = h.abs(), dy.double().abs()
    g = dya if w is None else dya * w.double().abs()
    e = row_error(x, rstd)
    a = g.mean(1, keepdim=True)
    c2 = (g * ha).mean(1, keepdim=True)
    b = (g * (1 + 2 * ha)).mean(1, keepdim=True)
    edx = rstd * e * (g + 2 * a + ha * (b + c2) + (1 + ha) * c2)
    edx = edx + half_step(dtype) * (dx.abs() + edx) + tiny(dtype)
    m = (x.shape[0] // 8 + 256) * U32
    edw = (dya * ((1 + ha) * e + ha * m)).sum(0)
    edw = edw + half_step(param_dtype) * (dw.abs() + edw) + tiny(param_dtype)
    edb = dya.sum(0) * m
    edb = edb + half_step(param_dtype) * (db.abs() + edb) + tiny(param_dtype)
    return (dx, edx), (dw, edw), (db, edb)


def grad_norm(tensors, norm_type=2.0) -> float:
    flat = torch.cat([t.double().reshape(-1) for t in tensors])
    if norm_type == 1.0:
        return float(flat.abs().sum())
    if norm_type == math.inf:
        return float(flat.abs().max()) if flat.numel() else 0.0
    return float((flat * flat).sum().sqrt())


def norm_bound(count: int) -> float:
    """Relative bound on a norm of `count` values: their sum (of terms of one
    sign) is off by at most the additions that a term passes through in
    float32, at most count / 512 + 64 (a CTA of 512 threads takes them all,
    or shares them; partial sums are joined in float64)."""
    return (count / 512 + 64) * U32


def scale_of(norm: float, max_norm: float) -> float:
    return min(1.0, max_norm / (norm + 1e-6))
