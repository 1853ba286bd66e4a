"""Float64 restatement of what stands between a layer's products, with error bounds:
the dropout's masks from the generator's definition, and the residual norm with its
gradients.

The bounds are worst cases, element by element, of an implementation in float32 that
rounds each result once. They are carried along with the values: an operation on
values that err by e1, e2 errs by what those errors make of its result and by half a
float32 step of it, 2^-24 relative, of its own. Sums over a row have at most
64 + cols / 256 additions on a value's way, sums over the rows any order.
"""

from __future__ import annotations

import torch

from .dense_torch import SUM_STEP, half_step, tiny

STEP = SUM_STEP / 2
MASK32 = 0xFFFFFFFF


def philox(counter: int, offset: int, seed: int) -> list[int]:
    """The four words of Philox4x32-10 at counter (64 bits each, low words first) under
    the key `seed`, in integers of any length."""
    c = [counter & MASK32, counter >> 32, offset & MASK32, offset >> 32]
    k = [seed & MASK32, seed >> 32]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [p1 >> 32 ^ c[1] ^ k[0], p1 & MASK32, p0 >> 32 ^ c[3] ^ k[1], p0 & MASK32]
        k = [(k[0] + 0x9E3779B9) & MASK32, (k[1] + 0xBB67AE85) & MASK32]
    return c


def kept(first: int, count: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """Which of the elements `first` to first + count - 1 dropout keeps."""
    border = round(p * 2.0**32)
    words = {}
    out = []
    for i in range(first, first + count):
        if i // 4 not in words:
            words[i // 4] = philox(i // 4, offset, seed)
        out.append(words[i // 4][i % 4] >= border)
    return torch.tensor(out, dtype=torch.bool)


def rounded(value, err, dtype):
    """(value, bound) of a result that is rounded to `dtype`."""
    u = half_step(dtype)
    return value, err * (1 + u) + u * value.abs() + tiny(dtype)


def dropout(x, keep, p, residual=None):
    """(value, bound) of the output."""
    out = torch.where(keep, x.double() / (1.0 - p), 0.0) if p < 1.0 else torch.zeros_like(x.double())
    err = 2 * SUM_STEP * out.abs()  # the scale's rounding and the product's
    if residual is not None:
        out = out + residual.double()
        err = err + SUM_STEP * out.abs()
    return rounded(out, err, x.dtype)


class Unit:
    """A row's norm: its unit row h with its error, the factor s with its relative one."""

    def __init__(self, x, kind, eps, x_err=0.0):
        cols = x.shape[-1]
        self.kind, self.depth = kind, 64 + cols // 256
        x = x.double()
        x_err = x_err + torch.zeros_like(x)
        if kind == "layer":
            # the mean as an offset from a base, corrected by the mean of the differences
            # (see layer_norm in dense_torch)
            mean = x.mean(-1, keepdim=True)
            c = x - mean
            offset = torch.minimum(mean.abs(), (mean - x[:, :1]).abs())
            e = STEP * (2 * c.abs() + 2 * offset + self.depth * c.abs().mean(-1, keepdim=True))
            e = e * (1 + 2.0**-10) + x_err + x_err.mean(-1, keepdim=True)
        else:
            c, e = x, x_err
        self.s = 1.0 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
        self.s_rel = ((c.abs() * e + e * e).mean(-1, keepdim=True) * self.s * self.s
                      + (self.depth + 8) * STEP)
        self.h = c * self.s
        self.h_err = (e * self.s * (1 + self.s_rel) + self.h.abs() * self.s_rel
                      + SUM_STEP * self.h.abs())

    def scaled(self, weight, bias):
        out = self.h * weight + bias
        err = (self.h_err * weight.abs()
               + 2 * SUM_STEP * ((self.h * weight).abs() + bias.abs()))
        return out, err

    def grad(self, v, v_err):
        """x's gradient from v of the unit row."""
        mh = (v * self.h).mean(-1, keepdim=True)
        mh_err = ((v.abs() * self.h_err + v_err * (self.h.abs() + self.h_err)).mean(-1, keepdim=True)
                  + (self.depth + 4) * STEP * (v * self.h).abs().mean(-1, keepdim=True))
        inner = v - self.h * mh
        inner_err = (v_err + self.h_err * (mh.abs() + mh_err) + self.h.abs() * mh_err
                     + 4 * SUM_STEP * (v.abs() + (self.h * mh).abs()))
        if self.kind == "layer":
            mv = v.mean(-1, keepdim=True)
            inner = inner - mv
            inner_err = (inner_err + v_err.mean(-1, keepdim=True)
                         + (self.depth + 4) * STEP * v.abs().mean(-1, keepdim=True)
                         + 4 * SUM_STEP * mv.abs())
        out = self.s * inner
        return out, (self.s * (1 + self.s_rel) * inner_err
                     + out.abs() * (self.s_rel + SUM_STEP))


def column_sum(value, err, dtype):
    total = value.sum(0)
    bound = err.sum(0) + (value.shape[0] + 2) * SUM_STEP * (value.abs() + err).sum(0)
    return rounded(total, bound, dtype)


def residual_norm(block, residual, weight=None, bias=None, *, norm="layer", eps=1e-5,
                  post_norm=None, post_weight=None, post_bias=None, gate=None,
                  residual_scale=1.0, p=0.0, keep=None, grad=None, grad_stream=None):
    """{name: (value, bound)} of the outputs and, with a gradient of one of them, the
    gradients of what is given. `keep`: the dropout's mask."""
    dtype = block.dtype
    vectors = {"weight": weight, "bias": bias, "gate": gate, "post_weight": post_weight,
               "post_bias": post_bias}
    wdtype = next((t.dtype for t in vectors.values() if t is not None), dtype)
    zero = torch.zeros(block.shape[-1], dtype=torch.float64, device=block.device)
    w, b, gt, pw, pb = (
        (zero if name.endswith("bias") else zero + 1.0) if t is None else t.double()
        for name, t in vectors.items())
    y, y_err = block.double(), torch.zeros_like(block, dtype=torch.float64)
    post = Unit(block, post_norm, eps) if post_norm is not None else None
    if post is not None:
        y, y_err = post.scaled(pw, pb)
    if keep is None:
        keep = torch.ones_like(block, dtype=torch.bool)
    scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    d = torch.where(keep, y * scale, 0.0)
    d_err = torch.where(keep, y_err * scale, 0.0) + 2 * SUM_STEP * d.abs()
    total = residual_scale * residual.double() + gt * d
    err = (gt.abs() * d_err + 2 * SUM_STEP * ((gt * d).abs() + total.abs()
                                              + (residual_scale * residual.double()).abs()))
    out = {"stream": rounded(total, err, dtype)}
    unit = Unit(total, norm, eps, err)
    out["normed"] = rounded(*unit.scaled(w, b), dtype)
    if grad is None and grad_stream is None:
        return out
    ds = torch.zeros_like(total) if grad_stream is None else grad_stream.double()
    ds_err = torch.zeros_like(total)
    if grad is not None:
        g = grad.double()
        v = g * w
        through, through_err = unit.grad(v, SUM_STEP * v.abs())
        ds = ds + through
        ds_err = through_err + SUM_STEP * ds.abs()
        if weight is not None:
            out["weight"] = column_sum(g * unit.h, g.abs() * unit.h_err, wdtype)
        if bias is not None:
            out["bias"] = column_sum(g, torch.zeros_like(g), wdtype)
    r = residual_scale * ds
    out["residual"] = rounded(r, abs(residual_scale) * ds_err + 2 * SUM_STEP * r.abs(), dtype)
    dt = torch.where(keep, ds * scale, 0.0)
    dt_err = torch.where(keep, ds_err * scale, 0.0) + 2 * SUM_STEP * dt.abs()
    if gate is not None:
        out["gate"] = column_sum(dt * y, dt_err * (y.abs() + y_err) + dt.abs() * y_err, wdtype)
    dy = dt * gt
    dy_err = dt_err * gt.abs() + SUM_STEP * dy.abs()
    if post is not None:
        if post_weight is not None:
            out["post_weight"] = column_sum(
                dy * post.h, dy_err * (post.h.abs() + post.h_err) + dy.abs() * post.h_err, wdtype)
        if post_bias is not None:
            out["post_bias"] = column_sum(dy, dy_err, wdtype)
        v = dy * pw
        dy, dy_err = post.grad(v, dy_err * pw.abs() + SUM_STEP * v.abs())
    out["block"] = rounded(dy, dy_err, dtype)
    return out
