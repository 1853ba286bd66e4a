"""What the dense operators' results may lose besides their one rounding, on the GPU
against float64: root mean squares over whole tensors, where a bound per element would
have to allow the worst order of a sum."""

import math

import pytest
import torch

from muspace_amd import layer_norm, linear
from oracle import dense_torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def rms(t):
    return float(t.double().square().mean().sqrt())


# ------------------------------------------------------ float32 products ---


@pytest.mark.parametrize(
    "size", [(9000, 72, 136), (20000, 64, 512), (9001, 203, 611), (6000, 520, 1030), (44446, 256, 96),
             (300, 256, 256), (1800, 1024, 256), (3, 203, 611), (1, 2048, 512)], ids=str)
@pytest.mark.parametrize("residual", [False, True])
def test_float32_products_have_float32_errors(size, residual):
    """Values with all their bits, in the kernels of many rows, of few results and of few rows:
    root mean squares, which two bfloat16 planes in place of three would exceed."""
    rows, inner, outer = size
    gen = torch.Generator(device=DEV).manual_seed(8)
    x, w, g = normal(gen, rows, inner), normal(gen, outer, inner), normal(gen, rows, outer)
    r = normal(gen, rows, outer) if residual else None
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = linear(xs, ws, residual=r)
    dx, dw = torch.autograd.grad(out, [xs, ws], g)
    y = x.double() @ w.double().t()
    for name, got, exact, k in (("out", out.detach(), y if r is None else y + r, inner),
                                ("grad_input", dx, g.double() @ w.double(), outer),
                                ("grad_weight", dw, g.double().t() @ x.double(), rows)):
        assert rms(got.double() - exact) <= dense_torch.product_rms(k) * rms(exact), name


# ------------------------------------------------------------ gelu's slope ---


def slope_values(codes):
    """The derivatives that 16-bit codes stand for: float16 numbers under 2^-5 (the negative
    ones after the positive), then steps of 2^-15, then NaN."""
    c = codes.to(torch.int64) & 0xFFFF
    tails = 0x2800
    bits = torch.where(c < tails, c, c - tails).clamp(0, tails - 1)
    tail = bits.to(torch.int16).view(torch.float16).double()
    tail = torch.where(c < tails, tail, -tail)
    step = (c - (2 * tails + 4230)).double() * 2.0**-15
    return torch.where(c < 2 * tails, tail, torch.where(c == 0xFFFF, math.nan, step))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_kept_slopes(native_lib, dtype):
    """Every kept derivative against the exact one, tails and crossings of zero included."""
    z = torch.cat([torch.linspace(-14.0, 14.0, 20001, device=DEV),
                   torch.linspace(-0.76, -0.74, 401, device=DEV),
                   torch.tensor([0.0, -0.0, 300.0, -300.0, math.inf, -math.inf, math.nan],
                                device=DEV)]).to(dtype)
    rows = z.numel()
    w = torch.ones((1, 1), dtype=dtype, device=DEV)
    out, kept = (torch.empty((rows, 1), dtype=dtype, device=DEV) for _ in range(2))
    native_lib.linear_forward(z.view(rows, 1), w, None, None, out, kept, 2)
    kept = kept.view(rows)
    values = kept.double() if dtype == torch.float32 else slope_values(kept.view(torch.int16))
    assert values[-1].isnan() and values[-7:-1].tolist() == [0.5, 0.5, 1.0, 0.0, 1.0, 0.0]
    values, exact = values[:-7], dense_torch.gelu_slope(z[:-7].double())
    # z is exact here. Relative to each term, z Phi' and Phi, the float32 evaluation of
    # exp(-z^2 / 2) errs by the roundings of z^2, of log2(e) / 2 and of their product, which
    # add up to 3 2^-24 z^2 / 2; 20 covers the other roundings. exp(-z^2 / 2) under the normal
    # numbers, 2^-126, may be zero: that moves z Phi' by less than |z| 2^-126 and Phi by less
    # than 2^-126.
    zd = z[:-7].double()
    density = torch.exp(-0.5 * zd * zd) / math.sqrt(2.0 * math.pi)
    terms = (zd * density).abs() + 0.5 * torch.special.erfc(-zd * math.sqrt(0.5))
    computed = terms * (20 + 1.5 * zd * zd) * 2.0**-24
    bound = computed + dense_torch.kept_slope_error(exact.abs() + computed, dtype)
    assert ((values - exact).abs() <= bound + (1 + zd.abs()) * 2.0**-126).all()


def test_gelu_keeps_the_digits_of_its_tails():
    """float32: relative to gelu's own value, however far below zero; the roundings of
    exp(-z^2 / 2) as above, 20 for the others."""
    z = torch.linspace(-13.0, 3.0, 30001, device=DEV)
    out = linear(z[:, None], torch.ones((1, 1), device=DEV), activation="gelu")[:, 0].double()
    zd = z.double()
    exact = dense_torch.gelu(zd)
    assert ((out - exact).abs() <= exact.abs() * (20 + 1.5 * zd * zd) * 2.0**-24 + 2.0**-126).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [(6000, 203, 611), (5000, 256, 512), (70, 96, 64)], ids=str)
def test_gelu_gradients_err_by_their_rounding(size, dtype):
    """The gradients' error is that of the formula in float32, rounded once: what is kept of
    the pre-activation in 16 bits adds less than 2%. A kept derivative is off by 2^-15 /
    sqrt(12) = 8.8e-6 (root mean square; smaller ones by less), dz as two numbers of a
    16-bit type by at most 2^-16 relative. Errors of single terms are independent, so
    that the products' relative error is of that size against dz's root mean square of
    about 0.6: under 2e-5, while the results' own rounding is 2e-4 in float16 and 1.6e-3
    in bfloat16. Squares add: under 1% more."""
    rows, inner, outer = size
    gen = torch.Generator(device=DEV).manual_seed(7)
    x = normal(gen, rows, inner).to(dtype)
    w = (normal(gen, outer, inner) / math.sqrt(inner)).to(dtype)
    b = (0.1 * normal(gen, outer)).to(dtype)
    g = normal(gen, rows, outer).to(dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(linear(*leaves, activation="gelu"), leaves, g)

    def formula(kind):
        xs, ws, bs, gs = (t.to(kind) for t in (x, w, b, g))
        z = xs @ ws.t() + bs
        dz = gs * (0.5 * torch.special.erfc(-z * math.sqrt(0.5))
                   + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))
        return dz @ ws, dz.t() @ xs, dz.sum(0)

    for name, got, plain, exact in zip(("grad_input", "grad_weight", "grad_bias"), grads,
                                       formula(torch.float32), formula(torch.float64)):
        if got.numel() < 4096:
            continue  # too few roundings for their root mean square to be known to 2%
        ratio = rms(got.double() - exact) / rms(plain.to(dtype).double() - exact)
        assert ratio <= 1.02, (name, ratio)


# -------------------------------------------------------------- layer norm ---


def plain_norm(x, w, b, eps, g, kind):
    """(y, dx, dw, db) in two passes over x in the floating-point type ``kind``."""
    x, w, b, g = (t.to(kind) for t in (x, w, b, g))
    c = x - x.mean(-1, keepdim=True)
    s = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    h, u = c * s, g * w
    dx = s * (u - u.mean(-1, keepdim=True) - h * (u * h).mean(-1, keepdim=True))
    return h * w + b, dx, (g * h).sum(0), g.sum(0)


@pytest.mark.parametrize("far", [0.0, 50.0], ids=["around_zero", "far_from_zero"])
@pytest.mark.parametrize("at", [0, 1, -1], ids=["first", "second", "last"])
@pytest.mark.parametrize("size", [10.0, 1e3, 1e5], ids=str)
@pytest.mark.parametrize("cols", [64, 256, 611, 1024, 4096, 20000])
def test_norm_of_rows_with_a_large_channel(cols, size, at, far):
    """A channel far from the others, wherever it lies, costs their results nothing: the
    error is that of the two-pass formula in float32. Both round each value's difference from
    the mean, and the mean, to float32; three times the plain error allows for the few
    roundings more of a sum in another order."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    rows = 400
    x = normal(gen, rows, cols) + far
    x[:, at] = size * (1.0 + 0.1 * normal(gen, rows))
    w, b = 1.0 + 0.2 * normal(gen, cols), 0.01 * normal(gen, cols)
    g = normal(gen, rows, cols)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    out = layer_norm(*leaves)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    others = [i for i in range(cols) if i != at % cols]
    exact = plain_norm(x, w, b, 1e-5, g, torch.float64)
    plain = plain_norm(x, w, b, 1e-5, g, torch.float32)
    for name, a, p, e in zip(("out", "grad_input", "grad_weight"), got, plain, exact):
        mine, theirs = (rms((t.double() - e)[..., others]) for t in (a, p))
        assert mine <= 3 * theirs, (name, mine / theirs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [8, 100, 256, 1000, 4096, 20000])
def test_norm_of_constant_and_nearly_constant_rows(cols, dtype):
    """Constant rows of any size give the bias itself and gradients without NaN; a step of
    one value's last bit is seen as such."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    info = torch.finfo(dtype)
    levels = torch.tensor([0.0, 3.3, -1000.0, info.max / 4, -info.max / 4, info.tiny], device=DEV)
    x = levels[:, None].expand(-1, cols).to(dtype)
    w, b = ((1.0 + 0.2 * normal(gen, cols)).to(dtype) for _ in range(2))
    xs = x.clone().requires_grad_()
    out = layer_norm(xs, w, b)
    assert torch.equal(out, b.expand_as(out))
    assert torch.autograd.grad(out, [xs], torch.ones_like(out))[0].isfinite().all()
    # rows of 1 with one value 1 + eps, first or last: h = sqrt(cols - 1) there and
    # -1 / sqrt(cols - 1) elsewhere, without eps
    near = torch.ones((2, cols), dtype=dtype, device=DEV)
    near[0, 0] = near[1, -1] = 1.0 + info.eps
    out = layer_norm(near, eps=0.0).double()
    expected = torch.full((2, cols), -1.0 / math.sqrt(cols - 1), dtype=torch.float64, device=DEV)
    expected[0, 0] = expected[1, -1] = math.sqrt(cols - 1)
    # each sum over the row errs by 2^-24 an addition on a value's way. In the first row the
    # others' mean lies eps from x0, and rounds by 2^-24 of that, as what is left of it
    # does: against sigma = eps / sqrt(cols), 2 sqrt(cols) 2^-24.
    slack = info.eps / 2 + (80 + cols / 128) * 2.0**-24
    bound = slack * expected.abs() + slack / math.sqrt(cols)
    bound[0] += 2 * math.sqrt(cols) * 2.0**-24
    assert ((out - expected).abs() <= bound).all()


def test_norm_of_values_whose_squares_overflow():
    """As in the formula: an infinite variance gives zeros, not values of any size."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    x = 1e30 * normal(gen, 5, 300)
    out = layer_norm(x)
    assert torch.equal(out, torch.zeros_like(out))
