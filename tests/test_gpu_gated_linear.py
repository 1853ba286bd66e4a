"""gated_linear on the GPU against float64."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from muspace_amd import gated_linear, get_last_dispatch_report
from oracle import dense_torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
GATES = [None, "relu", "gelu", "silu", "sigmoid"]
DEV = "cuda"


def make(rows, inner, hidden, dtype, *, bias=True, seed=0, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    x = normal(rows, inner).to(dtype)
    w = (size * normal(2 * hidden, inner) / math.sqrt(max(inner, 1))).to(dtype)
    b = normal(2 * hidden).to(dtype) if bias else None
    return x, w, b, normal(rows, hidden).to(dtype)


def assert_within(actual, expected, bound, what):
    assert actual.shape == expected.shape, what
    error = (actual.double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((error / bound.clamp_min(1e-300)).max())} of the bound")


def step(x, w, b, g, activation):
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b) if t is not None]
    out = gated_linear(leaves[0], leaves[1], leaves[2] if b is not None else None,
                       activation=activation)
    return [out.detach(), *torch.autograd.grad(out, leaves, g)]


def check(x, w, b, g, activation="silu"):
    got = step(x, w, b, g, activation)
    assert get_last_dispatch_report().selected_backend == "hip"
    results, bounds = dense_torch.gated_linear(x, w, b, activation, g)
    for name, a, e, t in zip(("out", "grad_input", "grad_weight", "grad_bias"), got, results, bounds):
        assert a.dtype == x.dtype
        assert_within(a, e, t, name)
    with torch.no_grad():  # the same call without a graph
        assert torch.equal(gated_linear(x, w, b, activation=activation), got[0])
    return got


SIZES = [
    (1, 1, 1), (1, 256, 256), (2, 8, 3), (3, 5, 7), (4, 100, 9), (5, 64, 40), (8, 70, 33),
    (17, 33, 65), (31, 64, 32), (33, 129, 40), (130, 256, 520), (300, 96, 64), (257, 203, 131),
    (1000, 40, 24),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_small_sizes(size, dtype):
    check(*make(*size, dtype))
    check(*make(*size, dtype, bias=False, seed=1), "gelu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(20011, 64, 32), (20000, 96, 80), (33001, 131, 77),
                                  (6000, 520, 515), (2049, 1024, 256), (513, 2048, 300),
                                  (4090, 1032, 1790), (16300, 1024, 448), (11700, 2056, 500)],
                         ids=str)
def test_larger_sizes(size, dtype):
    check(*make(*size, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", GATES)
@pytest.mark.parametrize("rows", [1, 3, 65, 5000])
def test_activations(rows, activation, dtype):
    # relu: sums that are float32 numbers, so that their side of zero is not their order's
    x, w, b, g = make(rows, 72, 56, dtype, seed=rows)
    if activation == "relu":
        x, w, b = ((t * 8).round() / 8 for t in (x, w, b))
    check(x, w, b, g, activation)


@pytest.mark.parametrize("activation", GATES)
def test_the_whole_range_of_a_gate(activation):
    """a over the reach of every tail, u one: the activation itself, and its derivative."""
    a = torch.cat([torch.linspace(-130, 130, 4001, device=DEV), torch.linspace(-2, 2, 1001, device=DEV),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30], device=DEV)])
    w = torch.tensor([[1.0], [0.0]], device=DEV)
    b = torch.tensor([0.0, 1.0], device=DEV)
    for x in (a[:, None], a[:4, None]):  # in tiles, and in few rows
        xs = x.clone().requires_grad_()
        out = gated_linear(xs, w, b, activation=activation)
        dx, = torch.autograd.grad(out, [xs], torch.ones_like(out))
        value, slope = dense_torch.gate(x.double(), activation)
        # a relative 16 float32 steps, and those of the exponent, |a| and its square at the worst;
        # a factor under float32's normal numbers, 2^-126, may be zero: silu is then up to
        # 87.4 * 2^-126 < 2^-119, where exp(z) passes 2^-126 (z = -87.3)
        near = dense_torch.SUM_STEP * (16 + (x.double().square() if activation == "gelu" else 0))
        assert_within(out.detach(), value, near * value.abs() + 2.0**-119, "value")
        # gelu's and silu's derivatives are sums of two terms that cancel at a zero near -0.75 and
        # -1.28: each term errs relatively to itself, the sum by as much as both
        z = x.double()
        terms = slope.abs()
        if activation == "gelu":
            terms = (0.5 * torch.special.erfc(-z * math.sqrt(0.5))
                     + z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
        elif activation == "silu":
            terms = torch.sigmoid(z) * (1 + z.abs() * torch.sigmoid(-z))
        assert_within(dx, slope, near * terms + 2.0**-119, "derivative")


def test_infinities_and_nan():
    """Limits of the gates at infinities; NaN stays, in its own results."""
    w = torch.tensor([[1.0], [0.0]], device=DEV)
    b = torch.tensor([0.0, 1.0], device=DEV)
    inf = math.inf
    x = torch.zeros((70, 1), device=DEV)
    for activation, top, low in ((None, inf, -inf), ("relu", inf, 0.0), ("gelu", inf, 0.0),
                                 ("silu", inf, 0.0), ("sigmoid", 1.0, 0.0)):
        # (an infinity times a weight of zero is NaN: the gate's half alone)
        for rows in (2, 70):
            xs = x[:rows].clone()
            big = torch.finfo(torch.float32).max
            xs[0], xs[1] = big, -big
            out = gated_linear(xs, w * 4, b, activation=activation)[:, 0]
            assert out[0] == top and out[1] == low, activation
            xs = xs.clone().requires_grad_()
            dx, = torch.autograd.grad(gated_linear(xs, w * 4, b, activation=activation).sum(), [xs])
            # (an infinite gate times the other half's weight of zero is NaN)
            assert dx[1].item() == 0.0 if activation is not None else dx[1].isnan()
            assert dx[0].item() == 0.0 if activation == "sigmoid" else dx[0].isnan()
            xs = x[:rows].clone()
            xs[1] = math.nan
            out = gated_linear(xs, w, b, activation=activation)
            assert out[1].isnan() and not out[0].isnan()


def test_values_past_the_type_become_infinities():
    x = torch.full((40, 8), 100.0, dtype=torch.float16, device=DEV, requires_grad=True)
    w = torch.full((8, 8), 10.0, dtype=torch.float16, device=DEV)
    out = gated_linear(x, w, activation=None)
    assert (out == math.inf).all()
    dx, = torch.autograd.grad(out, [x], torch.full_like(out, 10.0))
    assert (dx == math.inf).all()


def rms(a, e):
    return float((a.double() - e).square().mean().sqrt() / e.square().mean().sqrt())


@pytest.mark.parametrize("dtype", DTYPES)
def test_precision(dtype):
    """Root mean squares. The output and the bias's gradient err by their own rounding; the
    products by theirs and that of da and du, two independent errors of one size: sqrt(2), 3% of
    room (384 sums scatter more: 4 deviations are 4 / sqrt(2 * 384), 14%). float32: what
    products of that many terms may lose, twice over for two in a row, and 8 steps of the
    activation."""
    x, w, b, g = make(8000, 256, 192, dtype, seed=5)
    got = step(x, w, b, g, "silu")
    results, _ = dense_torch.gated_linear(x, w, b, "silu", g)
    for i, (a, e) in enumerate(zip(got, results)):
        own = rms(e.to(dtype), e)
        if dtype == torch.float32:
            limit = dense_torch.product_rms(256) + dense_torch.product_rms(8000) + 8 * 2.0**-24
        else:
            limit = own * (1.03, 1.03 * math.sqrt(2), 1.03 * math.sqrt(2), 1.14)[i]
        assert rms(a, e) <= limit, (i, rms(a, e), own)


def test_single_gradients_and_repeats():
    x, w, b, g = make(30000, 96, 80, torch.bfloat16)
    every = step(x, w, b, g, "silu")
    for a, e in zip(step(x, w, b, g, "silu"), every):
        assert torch.equal(a, e)
    for i in range(3):
        tensors = [t.clone() for t in (x, w, b)]
        tensors[i].requires_grad_()
        grad, = torch.autograd.grad(gated_linear(*tensors), [tensors[i]], g)
        assert torch.equal(grad, every[1 + i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype):
    for shape, hidden in (((0, 20), 6), ((2, 0, 5), 6), ((3, 0), 6), ((3, 20), 0), ((0,), 6)):
        xs, ws, bs = (torch.ones(s, dtype=dtype, device=DEV, requires_grad=True)
                      for s in (shape, (2 * hidden, shape[-1]), (2 * hidden,)))
        out = gated_linear(xs, ws, bs, activation=None)
        assert out.shape == (*shape[:-1], hidden)
        dx, dw, db = torch.autograd.grad(out, [xs, ws, bs], torch.ones_like(out))
        assert dx.shape == shape and not dw.any() and not dx.any()
        if out.numel():  # no inputs: a and u are the biases
            assert (out == 1).all() and (db == out.numel() // hidden).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner", [64, 45])
def test_unaligned_strided_and_negated(inner, dtype):
    x, w, b, g = make(200, inner, 40, dtype)
    results, bounds = dense_torch.gated_linear(x, w, b, "silu", g)

    def shifted(t):
        buffer = torch.full((t.numel() + 9,), math.nan, dtype=t.dtype, device=DEV)
        view = buffer[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    strided = [torch.stack([t, t], -1)[..., 0] for t in (x, w, b, g)]
    for tensors in ([shifted(t) for t in (x, w, b, g)], strided,
                    [x.t().contiguous().t(), w.t().contiguous().t(), b, g.t().contiguous().t()],
                    [torch._neg_view(-t) for t in (x, w, b, g)]):
        leaves = [t.detach().requires_grad_() for t in tensors[:3]]
        out = gated_linear(*leaves)
        for a, e, t in zip([out.detach(), *torch.autograd.grad(out, leaves, tensors[3])], results, bounds):
            assert_within(a, e, t, "strided")
    with torch.no_grad():
        flat = gated_linear(x, w, b)
        assert torch.equal(gated_linear(x.view(2, 5, 20, inner), w, b).view(200, 40), flat)
        assert_within(gated_linear(x[7], w, b), results[0][7], bounds[0][7], "one row")


def test_large_offsets():
    """More than 2^31 results: 64-bit offsets of rows, of da and du too."""
    rows, hidden = 2**20 + 77, 2056
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device=DEV)
    x[-300:] = torch.randn((300, 8), device=DEV).to(x.dtype)
    w = torch.randn((2 * hidden, 8), device=DEV).to(x.dtype)
    xs = x.clone().requires_grad_()
    out = gated_linear(xs, w)
    assert out.numel() > 2**31
    g = torch.zeros_like(out)
    g[-300:] = 1.0
    dx, = torch.autograd.grad(out, [xs], g)
    results, bounds = dense_torch.gated_linear(x[-300:], w, None, "silu", g[-300:])
    assert_within(out[-300:].detach(), results[0], bounds[0], "out")
    assert_within(dx[-300:], results[1], bounds[1], "grad_input")
    assert not dx[:-300].any()


def test_gradients_against_differences():
    x, w, b, g = make(40, 24, 18, torch.float32, seed=2)
    for activation in ("silu", "gelu", "sigmoid", None):
        grads = step(x, w, b, g, activation)[1:]
        gen = torch.Generator(device=DEV).manual_seed(3)
        h = 1e-4
        for i, grad in enumerate(grads):
            tensors = [t.double() for t in (x, w, b)]
            d = torch.randn(tensors[i].shape, generator=gen, device=DEV, dtype=torch.float64)

            def loss(sign):
                moved = list(tensors)
                moved[i] = moved[i] + sign * h * d
                return (dense_torch.gated_linear(*moved, activation)[0][0] * g.double()).sum()

            difference = (loss(1) - loss(-1)) / (2 * h)
            # float32 sums of at most 40 terms; differences err by h^2 times a third derivative
            slack = 400 * dense_torch.SUM_STEP * float((grad.double().abs() * d.abs()).sum()) + 1e-4
            assert abs(float((grad.double() * d).sum() - difference)) <= slack


def test_refused_on_the_device():
    x, w, b, _ = make(8, 16, 6, torch.float32)
    for call, error, message in (
            (lambda: gated_linear(x, w.cpu()), RuntimeError, "weight must be a ROCm device tensor"),
            (lambda: gated_linear(x, w, b.cpu()), RuntimeError, "bias must be a ROCm device tensor"),
            (lambda: gated_linear(x.double(), w), TypeError, "input must be"),
            (lambda: gated_linear(x, w[:11]), ValueError, "weight must be"),
            (lambda: gated_linear(x, w.half()), TypeError, "weight must be"),
            (lambda: gated_linear(x, w, b[:6]), ValueError, "bias must be"),
            (lambda: gated_linear(x, w, activation="tanh"), ValueError, "activation must be"),
            (lambda: gated_linear(x, w, backend="none"), RuntimeError, "unknown backend"),
            (lambda: torch.func.vmap(lambda t: gated_linear(t, w))(x.view(2, 4, 16)), RuntimeError, ""),
            (lambda: torch.jit.trace(lambda t: gated_linear(t, w), (x,)), RuntimeError, "cannot be traced")):
        with pytest.raises(error, match=message):
            call()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
            gated_linear(x, forward_ad.make_dual(w, w))
    xs = x.clone().requires_grad_()
    first, = torch.autograd.grad(gated_linear(xs, w).square().sum(), [xs], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate gated_linear twice"):
        first.sum().backward()


def test_recomputed_blocks():
    from torch.utils.checkpoint import checkpoint

    x, w, b, g = make(500, 64, 96, torch.bfloat16)

    def run(call):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        out = call(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = run(gated_linear)
    with torch.autograd.graph.save_on_cpu():
        offloaded = run(gated_linear)
    for got in (run(lambda *a: checkpoint(gated_linear, *a, use_reentrant=False)), offloaded):
        for a, e in zip(got, want):
            assert torch.equal(a, e)


@pytest.mark.parametrize("rows", [1, 300, 9000])
def test_streams_and_captured_steps(rows):
    """On another stream, and captured and replayed with eager work in between."""
    x, w, b, g = make(rows, 96, 80, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def run():
        out = gated_linear(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
    torch.cuda.current_stream().wait_stream(stream)
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for replay in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(x.shape, device=DEV) + replay)
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        for a, e in zip(got, run()):
            assert torch.equal(a, e)


WIDE_ROWS = [(1, 1024, 28672), (1, 2048, 23040), (2, 1024, 27784), (4, 1024, 28672), (5, 1024, 28672)]


@pytest.mark.parametrize("size", WIDE_ROWS, ids=str)
def test_few_rows_of_a_wide_layer(size):
    check(*make(*size, torch.bfloat16))


@pytest.mark.parametrize("size", [*WIDE_ROWS, (1, 9, 7), (3, 64, 24), (33, 40, 17), (300, 256, 512),
                                  (4096, 1024, 1792)], ids=str)
def test_nothing_is_written_past_the_workspace(native_lib, size):
    rows, inner, hidden = size
    x, w, b, g = make(*size, torch.bfloat16)
    need = native_lib.raw("gated_linear_backward_workspace_size")(2, rows, inner, hidden, 1, 1, 1)
    # as much again behind it, or the sums of twice 256 rows, whichever is more
    behind = max(need, 4 * 2 * hidden * 4)
    space = torch.full((need + behind,), 0x5A, dtype=torch.uint8, device=DEV)
    assert space.data_ptr() % 256 == 0
    grads = [torch.empty_like(t) for t in (x, w, b)]
    assert native_lib.raw("gated_linear_backward")(
        g.data_ptr(), 2, x.data_ptr(), w.data_ptr(), b.data_ptr(), *(t.data_ptr() for t in grads),
        rows, inner, hidden, 3, space.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    assert (space[need:] == 0x5A).all()
    for got, want in zip(grads, step(x, w, b, g, "silu")[1:]):
        assert torch.equal(got, want)


@pytest.mark.parametrize("size", [(128, 1024, 28672), (130, 1024, 28672), (300, 1024, 28672), (60000, 1024, 64),
                                  (60000, 1024, 68), (60000, 1024, 160)], ids=str)
def test_borders_of_large_tiles(size):
    check(*make(*size, torch.bfloat16))


def gate_bounds(z, activation, dtype):
    """(value, derivative, bounds of their errors before they are rounded) of a gate in a type.

    16 bits: silu's and sigmoid's factors are off by a relative 2^-24 (1.3 |z| + 32), the
    exponent's rounding and a few of operations; float32 and the other gates as in
    test_the_whole_range_of_a_gate. The products keep silu to |z| steps of 2^-149; sigmoid and
    its derivative may be zero where they are under 2^-126, and gelu's under 2^-119."""
    value, slope = dense_torch.gate(z, activation)
    near = dense_torch.SUM_STEP * (16 + (z.square() if activation == "gelu" else 0))
    if dtype != torch.float32 and activation in ("silu", "sigmoid"):
        near = 2.0**-24 * (1.3 * z.abs() + 40)
    terms = slope.abs()
    if activation == "gelu":
        terms = (0.5 * torch.special.erfc(-z * math.sqrt(0.5))
                 + z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    elif activation == "silu":
        terms = torch.sigmoid(z) * (1 + z.abs() * torch.sigmoid(-z))
    floor = {"silu": (z.abs() + 1) * 2.0**-149, "sigmoid": 2.0**-126, "gelu": 2.0**-119}.get(activation, 0)
    # (2 near: the derivative has both factors, the sigmoid's their product)
    return value, slope, near * value.abs() + floor, 2 * near * terms + floor


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", GATES)
def test_the_tails_of_a_gate_in_every_type(activation, dtype):
    """As far as the type's numbers reach: a saturated sigmoid's derivative and silu's far left
    keep their relative accuracy."""
    a = torch.cat([torch.linspace(-130, 130, 4001, device=DEV), torch.linspace(-2, 2, 1001, device=DEV),
                   torch.linspace(-95, -86, 181, device=DEV)]).to(dtype)
    w = torch.tensor([[1.0], [0.0]], dtype=dtype, device=DEV)
    b = torch.tensor([0.0, 1.0], dtype=dtype, device=DEV)
    for x in (a[:, None], a[-4:, None], a[-40:, None]):  # in tiles, few rows, few results
        xs = x.clone().requires_grad_()
        out = gated_linear(xs, w, b, activation=activation)
        dx, = torch.autograd.grad(out, [xs], torch.ones_like(out))
        value, slope, value_err, slope_err = gate_bounds(x.double(), activation, dtype)
        for got, e, err in ((out.detach(), value, value_err), (dx, slope, slope_err)):
            # rounded once
            u, small = dense_torch.half_step(dtype), dense_torch.tiny(dtype)
            assert_within(got, e, err * (1 + u) + u * e.abs() + small, activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 70, 5000])
def test_limits_and_nan_in_every_type(rows, dtype):
    """The limits of the gates and of their derivatives at infinities; NaN stays in its results."""
    inf = math.inf
    w = torch.ones((2, 1), dtype=dtype, device=DEV)
    # the other half is a constant: its weight is zero, and no infinity meets it in the products
    w[1] = 0.0
    b = torch.tensor([inf, 1.0], dtype=dtype, device=DEV)
    x = torch.zeros((rows, 1), dtype=dtype, device=DEV)
    for activation, top, low, above, below in (
            (None, inf, -inf, 1.0, 1.0), ("relu", inf, 0.0, 1.0, 0.0), ("gelu", inf, 0.0, 1.0, 0.0),
            ("silu", inf, 0.0, 1.0, 0.0), ("sigmoid", 1.0, 0.0, 0.0, 0.0)):
        for sign, value, slope in ((1.0, top, above), (-1.0, low, below)):
            bias = (b * torch.tensor([sign, 1.0], dtype=dtype, device=DEV)).requires_grad_()
            out = gated_linear(x, w, bias, activation=activation)
            assert (out == value).all(), (activation, sign)
            db, = torch.autograd.grad(out, [bias], torch.ones_like(out))
            # (5000 rounds to the bfloat16 number 4992)
            assert db[0] == torch.tensor(slope * rows).to(dtype), (activation, sign)
        xs = x.clone()
        xs[1] = math.nan
        out = gated_linear(xs, w, activation=activation)
        assert out[1].isnan() and not out[0].isnan()
        # and in the gate's own derivative
        xs.requires_grad_()
        dx, = torch.autograd.grad(gated_linear(xs, w, activation=activation), [xs],
                                  torch.ones((rows, 1), dtype=dtype, device=DEV))
        assert dx[1].isnan() and not dx[0].isnan()
