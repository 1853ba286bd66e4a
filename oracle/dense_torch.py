"""Float64 restatement of the layer's dense operators, with error bounds.

``linear`` and ``layer_norm`` with their gradients in float64 from the formulas,
and the 8-bit checkpoint in exact arithmetic. The bounds are worst cases, element
by element, of an implementation that sums in float32 in any order and rounds
each result once: a sum of n products errs by at most (n + 2) 2^-23 times the sum
of their magnitudes (two float32 roundings of 2^-24 per term), a result by half a
step of its type more.
"""

from __future__ import annotations

import math

import torch

SUM_STEP = 2.0**-23


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def product_rms(k: int) -> float:
    """What the error of a float32 product of k random terms of either sign may be, as root
    mean squares over the result and relative to the result's own. A rounding errs by 0.4
    2^-24 of the partial sum; after i terms that is sqrt(i / k) of the result. Three planes
    take six products a term, each rounded into the sum at the worst: 0.4 2^-24 sqrt(6 k
    / 2). The parts of a long sum are added apart: 1024 terms at the most count. 4 2^-24
    are for the operands' planes, the parts' sum and the result."""
    return 2.0**-24 * (0.7 * math.sqrt(min(k, 1024)) + 4)


def gelu(z):
    return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))


def gelu_slope(z):
    return (0.5 * torch.special.erfc(-z * math.sqrt(0.5))
            + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))


def kept_slope_error(slope, dtype):
    """Of gelu's derivatives of up to these magnitudes as a backward keeps them: float32
    rounds them; 16 bits hold steps of 2^-15 from 2^-5 on, below that float16 numbers
    (subnormal under 2^-14, in steps of 2^-24)."""
    if dtype == torch.float32:
        return 2.0**-24 * slope
    return torch.where(slope < 2.0**-5, torch.maximum(2.0**-11 * slope, slope.new_tensor(2.0**-25)),
                       slope.new_tensor(2.0**-16))


def checkpoint(x):
    """(codes, scale bytes, restored values) of a finite or non-finite x [rows, cols]."""
    dtype = x.dtype
    low = -24 if dtype == torch.float16 else -126
    rows, cols = x.shape
    padded = (cols + 31) // 32 * 32
    values = torch.zeros((rows, padded), dtype=torch.float64, device=x.device)
    values[:, :cols] = x.double()
    blocks = values.view(rows, -1, 32)
    finite = torch.isfinite(blocks).all(-1, keepdim=True)
    top = torch.where(finite, blocks, 0.0).abs().amax(-1, keepdim=True)
    exponent = torch.full_like(top, float(low))
    # step up from the lowest exponent: no logarithm to round
    for e in range(low, 123):
        exponent = torch.where(top > 127.0 * 2.0**e, float(e + 1), exponent)
    scale = torch.exp2(exponent)
    codes = torch.round(blocks / scale)
    past = codes.abs() * scale > torch.finfo(dtype).max
    codes = torch.where(past, codes.sign() * 63.0, codes)
    codes = torch.where(finite, codes, 1.0)
    restored = torch.where(finite, codes * scale, math.nan).view(rows, padded)[:, :cols]
    scales = torch.where(finite, exponent + 127.0, 255.0).view(rows, -1)
    return codes.view(rows, padded).to(torch.int8), scales.to(torch.uint8), restored


def linear(x, weight, bias, activation, residual, grad=None, kept=None):
    """([results], [bounds]): y, and with ``grad`` dx, dW, db. ``kept`` [rows, in]
    float64 replaces x in dW (an 8-bit checkpoint)."""
    dtype, u, small = x.dtype, half_step(x.dtype), tiny(x.dtype)
    x, w = x.double(), weight.double()
    rows, inner = x.shape
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device)
    if bias is not None:
        b = bias.double()
    z = x @ w.t() + b
    z_err = (inner + 2) * SUM_STEP * (x.abs() @ w.abs().t() + b.abs())
    if activation == "relu":
        y, slope, y_err = z.clamp_min(0.0), (z > 0).double(), z_err
    elif activation == "gelu":
        # |slope| < 1.13; erf, two products and a sum: 8 float32 steps of z
        y, slope = gelu(z), gelu_slope(z)
        y_err = 1.13 * z_err + 8 * SUM_STEP * z.abs()
    else:
        y, slope, y_err = z, torch.ones_like(z), z_err
    if residual is not None:
        y = y + residual.double()
        y_err = y_err + SUM_STEP * y.abs()
    results, bounds = [y], [y_err * (1 + u) + u * y.abs() + small]
    if grad is None:
        return results, bounds
    g = grad.double()
    dz = g * slope
    dz_err = torch.zeros_like(dz)
    if activation == "gelu":
        # the slope (|slope'| < 0.8) is a float32 function of z and kept in the type's size;
        # dz is held to twice the type's bits (float32's at most)
        slope_err = 0.8 * z_err + 16 * SUM_STEP
        dz_err = g.abs() * (slope_err + kept_slope_error(slope.abs() + slope_err, dtype))
        dz_err = dz_err + max(u * u, SUM_STEP) * dz.abs() + small
    dx = dz @ w
    dx_err = (dz_err @ w.abs()
              + (w.shape[0] + 2) * SUM_STEP * ((dz.abs() + dz_err) @ w.abs()))
    rest = x if kept is None else kept
    dw = dz.t() @ rest
    dw_err = (dz_err.t() @ rest.abs()
              + (rows + 2) * SUM_STEP * ((dz.abs() + dz_err).t() @ rest.abs()))
    db = dz.sum(0)
    db_err = dz_err.sum(0) + (rows + 2) * SUM_STEP * (dz.abs() + dz_err).sum(0)
    for value, err in ((dx, dx_err), (dw, dw_err), (db, db_err)):
        results.append(value)
        bounds.append(err * (1 + u) + u * value.abs() + small)
    return results, bounds


def layer_norm(x, weight, bias, eps, grad=None):
    """([results], [bounds]): y, and with ``grad`` dx, dw, db (of the weight's type).

    The bounds are of a two-pass form whose sums over a row have at most D additions on
    any value's way (a part of the row per lane, then a tree), D = 64 + cols / 256. c = (x -
    base) - offset, base + offset the mean and |offset| <= min(|mean|, |mean - x0|), x0
    the row's first value. x - base, the offset and c round once each, and the offset
    is corrected by the mean of c, so that c errs by e = 2^-24 (2 |c| + 2 |offset| + D mean|c|),
    whatever the row's largest value. s errs by a relative mean(|c| e) / sigma^2 from
    c (sigma = 1 / s) and (D + 8) 2^-24 from its own sums and operations.
    """
    dtype, u, small = x.dtype, half_step(x.dtype), tiny(x.dtype)
    wdtype = weight.dtype if weight is not None else dtype
    rows, cols = x.shape
    x = x.double()
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    sigma = (c.square().mean(-1, keepdim=True) + eps).sqrt()
    s = 1.0 / sigma
    step, depth = SUM_STEP / 2, 64 + cols // 256
    offset = torch.minimum(mean.abs(), (mean - x[:, :1]).abs())
    e = step * (2 * c.abs() + 2 * offset + depth * c.abs().mean(-1, keepdim=True)) * (1 + 2.0**-10)
    s_rel = (c.abs() * e + e * e).mean(-1, keepdim=True) * s * s + (depth + 8) * step
    h = c * s
    h_err = e * s * (1 + s_rel) + h.abs() * s_rel + SUM_STEP * h.abs()
    y = h * w + b
    y_err = h_err * w.abs() + 2 * SUM_STEP * (h.abs() * w.abs() + b.abs())
    results, bounds = [y], [y_err * (1 + u) + u * y.abs() + small]
    if grad is None:
        return results, bounds
    g = grad.double()
    v = g * w
    mv, mh = v.mean(-1, keepdim=True), (v * h).mean(-1, keepdim=True)
    inner = v - mv - h * mh
    mv_err = (depth + 4) * step * v.abs().mean(-1, keepdim=True)
    mh_err = ((v.abs() * h_err).mean(-1, keepdim=True)
              + (depth + 4) * step * (v * h).abs().mean(-1, keepdim=True))
    inner_err = (mv_err + h_err * (mh.abs() + mh_err) + h.abs() * mh_err
                 + 4 * SUM_STEP * (v.abs() + mv.abs() + (h * mh).abs()))
    dx = s * inner
    dx_err = s * (1 + s_rel) * inner_err + dx.abs() * (s_rel + SUM_STEP)
    results.append(dx)
    bounds.append(dx_err * (1 + u) + u * dx.abs() + small)
    u, small = half_step(wdtype), tiny(wdtype)
    dw, db = (g * h).sum(0), g.sum(0)
    dw_err = ((g.abs() * h_err).sum(0)
              + (rows + 2) * SUM_STEP * (g.abs() * (h.abs() + h_err)).sum(0))
    db_err = (rows + 2) * SUM_STEP * g.abs().sum(0)
    for value, err in ((dw, dw_err), (db, db_err)):
        results.append(value)
        bounds.append(err * (1 + u) + u * value.abs() + small)
    return results, bounds
