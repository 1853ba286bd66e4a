"""layer_norm on the GPU against float64."""

import math

import pytest
import torch

from muspace_amd import get_last_dispatch_report, layer_norm
from oracle import dense_torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"
EPS = 1e-5


def make(rows, cols, dtype, weight_dtype=None, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    wdtype = dtype if weight_dtype is None else weight_dtype
    spread = torch.exp(0.5 * torch.randn(cols, generator=gen, device=DEV))
    x = (torch.randn((rows, cols), generator=gen, device=DEV) * spread + 0.5).to(dtype)
    w = (1.0 + 0.3 * torch.randn(cols, generator=gen, device=DEV)).to(wdtype)
    b = (0.3 * torch.randn(cols, generator=gen, device=DEV)).to(wdtype)
    g = torch.randn((rows, cols), generator=gen, device=DEV).to(dtype)
    return x, w, b, g


def assert_within(actual, expected, bound, what):
    assert actual.shape == expected.shape, what
    error = (actual.double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((error / bound.clamp_min(1e-300)).max())} of the bound")


def check(x, w, b, g, eps=EPS):
    leaves = [None if t is None else t.detach().clone().requires_grad_() for t in (x, w, b)]
    out = layer_norm(*leaves, eps=eps)
    assert get_last_dispatch_report().selected_backend == "hip"
    assert out.dtype == x.dtype
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(out, wanted, g)
    results, bounds = dense_torch.layer_norm(x, w, b, eps, g)
    names = ["out", "grad_input"] + ["grad_weight"] * (w is not None) + ["grad_bias"] * (b is not None)
    picks = [0, 1] + [2] * (w is not None) + [3] * (b is not None)
    for name, i, a in zip(names, picks, [out.detach(), *grads]):
        assert_within(a, results[i], bounds[i], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=eps), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    ("rows", "cols"),
    [(1, 1), (1, 2), (3, 7), (5, 64), (33, 128), (64, 129), (300, 256), (77, 255), (1, 512),
     (130, 513), (41, 1024), (19, 1500), (12, 2048), (9, 2051), (5, 4096), (4, 4100), (3, 9000),
     (3, 16384), (2, 16400), (2, 40001), (20000, 96), (40013, 256), (3000, 611)])
def test_sizes(rows, cols, dtype):
    check(*make(rows, cols, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [40, 203, 256, 1024, 3000, 20000])
def test_float32_weights_of_a_16_bit_input(cols, dtype):
    check(*make(130, cols, dtype, torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_optional_weight_and_bias(dtype):
    x, w, b, g = make(90, 200, dtype)
    check(x, None, None, g)
    check(x, w, None, g)
    check(x, None, b, g)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_far_from_zero_and_constant_rows(dtype):
    x, w, b, g = make(64, 256, dtype)
    x[:32] = x[:32] * (0.02 if dtype != torch.float32 else 1e-3) + 100.0
    x[40] = 3.3
    x[41] = 0.0
    x[42] = torch.finfo(dtype).max / 4
    out = layer_norm(x, w, b)
    # c = 0 exactly: the output is the bias
    for row in (40, 41, 42):
        assert torch.equal(out[row], b)
    keep = [i for i in range(64) if i not in (40, 41, 42)]
    check(x[keep], w, b, g[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinity_and_nan_stay_in_their_rows(dtype):
    x, w, b, g = make(50, 256, dtype)
    clean = layer_norm(x, w, b)
    x[7, 5], x[8, 255], x[9, 0] = math.nan, math.inf, -math.inf
    out = layer_norm(x, w, b)
    for row in (7, 8, 9):
        assert out[row].isnan().all()
    rest = [i for i in range(50) if i not in (7, 8, 9)]
    assert torch.equal(out[rest], clean[rest])
    xs = x.clone().requires_grad_()
    dx, = torch.autograd.grad(layer_norm(xs, w, b), [xs], g)
    assert dx[rest].isfinite().all() and dx[[7, 8, 9]].isnan().all()


def test_eps():
    x, w, b, g = make(40, 96, torch.float32)
    for eps in (0.0, 1e-12, 1e-3, 10.0):
        check(x, w, b, g, eps)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype):
    for shape in ((0, 64), (3, 0), (2, 0, 5), (0, 20000)):
        x = torch.empty(shape, dtype=dtype, device=DEV).requires_grad_()
        w = torch.ones(shape[-1], dtype=dtype, device=DEV).requires_grad_()
        b = torch.ones(shape[-1], dtype=dtype, device=DEV).requires_grad_()
        out = layer_norm(x, w, b)
        assert out.shape == shape
        dx, dw, db = torch.autograd.grad(out, [x, w, b], torch.empty_like(out))
        assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 100])
def test_unaligned_and_strided(cols, dtype):
    x, w, b, g = make(120, cols, dtype)
    results, bounds = dense_torch.layer_norm(x, w, b, EPS, g)

    def shifted(t):
        buffer = torch.full((t.numel() + 9,), math.nan, dtype=t.dtype, device=DEV)
        view = buffer[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    for xs, ws, bs, gs in ((*(shifted(t) for t in (x, w, b, g)),),
                           (x.t().contiguous().t(), torch.stack([w, w], -1)[:, 0],
                            torch.stack([b, b], -1)[:, 0], torch.cat([g, g], -1)[:, :cols])):
        leaves = [t.requires_grad_() for t in (xs, ws, bs)]
        out = layer_norm(*leaves)
        got = [out.detach(), *torch.autograd.grad(out, leaves, gs)]
        for a, e, t in zip(got, results, bounds):
            assert_within(a, e, t, "strided")


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dimensions_and_one_dimension(dtype):
    x, w, b, _ = make(24, 80, dtype)
    flat = layer_norm(x, w, b)
    assert torch.equal(layer_norm(x.view(2, 3, 4, 80), w, b).view(24, 80), flat)
    assert torch.equal(layer_norm(x[5], w, b), flat[5])


def test_single_gradients_and_repeats():
    x, w, b, g = make(30000, 192, torch.bfloat16)

    def grads(*which):
        tensors = [t.clone() for t in (x, w, b)]
        for i in which:
            tensors[i].requires_grad_()
        return torch.autograd.grad(layer_norm(*tensors), [tensors[i] for i in which], g)

    every = grads(0, 1, 2)
    for _ in range(2):
        for a, e in zip(grads(0, 1, 2), every):
            assert torch.equal(a, e)
    for i in range(3):
        assert torch.equal(grads(i)[0], every[i])


def test_large_offsets():
    """More than 2^31 values: 64-bit row offsets."""
    rows, cols = 2**20 + 5, 2056
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2**31
    x.zero_()
    gen = torch.Generator(device=DEV).manual_seed(0)
    x[-40:] = torch.randn((40, cols), generator=gen, device=DEV).to(x.dtype)
    out = layer_norm(x)
    results, bounds = dense_torch.layer_norm(x[-40:], None, None, EPS)
    assert_within(out[-40:], results[0], bounds[0], "large")


def test_gradients_against_differences():
    x, w, b, g = make(40, 72, torch.float32, seed=2)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    gen = torch.Generator(device=DEV).manual_seed(3)
    h = 1e-4
    for i, grad in enumerate(grads):
        tensors = [t.double() for t in (x, w, b)]
        d = torch.randn(tensors[i].shape, generator=gen, device=DEV, dtype=torch.float64)

        def loss(sign):
            moved = list(tensors)
            moved[i] = moved[i] + sign * h * d
            return (dense_torch.layer_norm(*moved, EPS)[0][0] * g.double()).sum()

        difference = (loss(1) - loss(-1)) / (2 * h)
        # float32 sums of at most 72 (dx) or 40 terms, of magnitudes up to a few times the
        # gradient's own; differences err by h^2 times a third derivative
        slack = 400 * dense_torch.SUM_STEP * float((grad.double().abs() * d.abs()).sum()) + 1e-4
        assert abs(float((grad.double() * d).sum() - difference)) <= slack


def test_refused_on_the_device():
    x, w, b, g = make(8, 16, torch.float32)
    with pytest.raises(RuntimeError, match="weight must be a ROCm device tensor"):
        layer_norm(x, w.cpu(), b.cpu())
    for args, kwargs, error, message in (
            ((x.double(),), {}, TypeError, "input must be"),
            ((x[0, 0],), {}, ValueError, "at least one dimension"),
            ((x, w[:3]), {}, ValueError, "weight must be"),
            ((x, w.half()), {}, TypeError, "weight must be"),
            ((x.half(), w, b.half()), {}, TypeError, "of one type"),
            ((x, w, torch.stack([b, b])), {}, ValueError, "bias must be"),
            ((x, w, b), {"eps": -1.0}, ValueError, "eps"),
            ((x, w, b), {"backend": "none"}, RuntimeError, "unknown backend")):
        with pytest.raises(error, match=message):
            layer_norm(*args, **kwargs)
    assert torch.equal(layer_norm(x, w, b, backend="musa"), layer_norm(x, w, b))


def test_tensor_level_entries(native_lib):
    """The library's checked entries on caller-owned tensors give the operator's results."""
    x, w, b, g = make(300, 200, torch.float16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want_out = layer_norm(*leaves)
    want = torch.autograd.grad(want_out, leaves, g)
    out, stats = torch.empty_like(x), torch.empty((300, 2), dtype=torch.float32, device=DEV)
    native_lib.layer_norm_forward(x, w, b, out, stats, EPS)
    assert torch.equal(out, want_out)
    got = [torch.full_like(t, math.nan) for t in (x, w, b)]
    native_lib.layer_norm_backward(g, x, w, stats, *got)
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    with pytest.raises(RuntimeError, match="statistics must have shape"):
        native_lib.layer_norm_forward(x, w, b, out, stats[:5], EPS)
    with pytest.raises(RuntimeError, match="weight must be float16"):
        native_lib.layer_norm_forward(x, w.double(), b, out, stats, EPS)
    with pytest.raises(RuntimeError, match="grad_bias must be float16"):
        native_lib.layer_norm_backward(g, x, w, stats, None, None, got[2].float())


def test_streams_and_captured_steps():
    """On another stream, and captured and replayed with eager work in between."""
    x, w, b, g = make(9000, 256, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def step():
        out = layer_norm(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    torch.cuda.current_stream().wait_stream(stream)
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(x.shape, device=DEV) + replay)
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        for a, e in zip(got, step()):
            assert torch.equal(a, e)
