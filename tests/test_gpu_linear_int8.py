"""linear_int8 and quantize_int8 on the GPU against exact integers and float64."""

import math

import pytest
import torch

from muspace_amd import get_last_dispatch_report, linear_int8, quantize_int8
from muspace_amd.ops import quantize_int8_pytorch
from oracle import dense_torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"


def make(rows, inner, outer, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    x = (normal(rows, inner) * torch.exp(0.5 * normal(inner))).to(dtype)
    w, s = quantize_int8(normal(outer, inner))
    return x, w, s, normal(outer).to(dtype), normal(rows, outer).to(dtype)


def assert_within(actual, expected, bound, what):
    assert actual.shape == expected.shape, what
    error = (actual.double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((error / bound.clamp_min(1e-300)).max())} of the bound")


def check(x, w, s, b, r, activation=None):
    out = linear_int8(x, w, s, b, activation=activation, residual=r)
    assert get_last_dispatch_report().selected_backend == "hip"
    assert out.dtype == x.dtype
    assert_within(out, *dense_torch.linear_int8(x, w, s, b, activation, r), "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 3, 15, 16, 17, 64, 100, 128, 256, 611, 1000, 2048, 4096, 5003,
                                  20000])
def test_quantize(cols, dtype):
    gen = torch.Generator(device=DEV).manual_seed(cols)
    info = torch.finfo(dtype)
    x = torch.randn((75, cols), generator=gen, device=DEV)
    x *= torch.exp2(torch.randint(-40, 12, (75, 1), generator=gen, device=DEV).float())
    x = x.to(dtype)
    x[0], x[1], x[2], x[3] = 0.0, info.max, -info.max, info.smallest_normal
    x[4] = info.smallest_normal / 4
    x[5, 0], x[6, cols - 1] = math.inf, math.nan
    x[7] = torch.arange(cols, device=DEV) % 128
    x[7, 0] = 127.0
    x[8] = torch.arange(cols, device=DEV) % 127 + 0.5  # ties
    x[8, 0] = -127.0
    codes, scales = quantize_int8(x)
    want, want_scales = dense_torch.quantize(x)
    assert torch.equal(codes, want)
    assert torch.equal(scales.nan_to_num(-1), want_scales.nan_to_num(-1))
    mine = quantize_int8(x.cpu())
    assert torch.equal(codes.cpu(), mine[0])
    buffer = torch.full((x.numel() + 9,), math.nan, dtype=dtype, device=DEV)
    buffer[1:1 + x.numel()].copy_(x.view(-1))
    for other in (buffer[1:1 + x.numel()].view(x.shape), x.t().contiguous().t(), torch._neg_view(-x)):
        assert torch.equal(quantize_int8(other)[0], codes)


SIZES = [
    (1, 1, 1), (1, 256, 256), (2, 8, 3), (3, 5, 7), (17, 33, 65), (31, 64, 32), (33, 129, 40),
    (130, 256, 520), (300, 96, 64), (257, 203, 131), (1000, 40, 24), (64, 2048, 100), (5, 5000, 17),
    (3, 131072, 5), (4, 12288, 33), (3, 12300, 33), (2, 24570, 40), (1, 49150, 20),
    (1, 4100, 500), (3, 2047, 19), (40, 2048, 70), (40, 2049, 70), (20011, 64, 32),
    (20000, 96, 160), (33001, 131, 77), (6000, 520, 1030), (2049, 1024, 256), (513, 2048, 300),
    (4090, 1040, 3580), (16300, 1024, 900),
    (11700, 4112, 1000), (24577, 256, 200), (24600, 64, 513), (30000, 240, 512), (25001, 3, 130),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, dtype):
    x, w, s, b, r = make(*size, dtype)
    check(x, w, s, b, r)
    check(x, w, s, b, None, "relu")
    check(x, w, s, None, r, "gelu")


def test_extreme_codes_and_sums():
    """Every code at its end over the longest sum, weights of -128 among them: exact."""
    x = torch.full((40, 131072), 3.0, device=DEV)
    w = torch.full((50, 131072), 127, dtype=torch.int8, device=DEV)
    w[7], w[8] = -128, -127
    s = torch.ones(50, device=DEV)
    out = linear_int8(x, w, s)
    check(x, w, s, None, None)
    top = float(torch.tensor(127.0 * 127 * 131072)) * float(quantize_int8(x[:1])[1])
    assert out[0, 0].item() == pytest.approx(top, rel=2.0**-23)
    assert (out[:, 7] < out[:, 8]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 50, 9000, 25000])
def test_infinity_and_nan_stay_in_their_rows(rows, dtype):
    x, w, s, b, r = make(rows, 200, 72, dtype)
    clean = linear_int8(x, w, s, b, residual=r)
    x[0, 5], x[1, 199] = math.nan, -math.inf
    out = linear_int8(x, w, s, b, residual=r)
    assert out[:2].isnan().all() and torch.equal(out[2:], clean[2:])
    assert linear_int8(x, w, s, activation="relu")[:2].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner", [64, 45, 7])
def test_unaligned_strided_and_negated(inner, dtype):
    x, w, s, b, r = make(200, inner, 40, dtype)
    want = linear_int8(x, w, s, b, residual=r)

    def shifted(t):
        buffer = torch.full((t.numel() + 9,), 99 if t.dtype == torch.int8 else math.nan, dtype=t.dtype,
                            device=DEV)
        view = buffer[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    for args in ([shifted(t) for t in (x, w, s, b, r)],
                 [torch.stack([t, t], -1)[..., 0] for t in (x, w, s, b, r)],
                 [x.t().contiguous().t(), w.t().contiguous().t(), s, b, r],
                 [torch._neg_view(-t) if t.is_floating_point() else t for t in (x, w, s, b, r)]):
        assert torch.equal(linear_int8(*args[:4], residual=args[4]), want)
    assert torch.equal(linear_int8(x.view(2, 5, 20, inner), w, s, b, residual=r.view(2, 5, 20, 40)),
                       want.view(2, 5, 20, 40))
    assert torch.equal(linear_int8(x[7], w, s, b, residual=r[7]), want[7])


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype):
    for shape, outer in (((0, 20), 6), ((2, 0, 5), 6), ((3, 0), 6), ((3, 20), 0), ((0,), 6)):
        x = torch.ones(shape, dtype=dtype, device=DEV)
        w, s = quantize_int8(torch.ones(outer, shape[-1], device=DEV))
        b = torch.ones(outer, dtype=dtype, device=DEV)
        out = linear_int8(x, w, s, b)
        assert out.shape == (*shape[:-1], outer)
        if shape[-1] == 0:
            assert (out == 1).all()


def test_large_offsets():
    """More than 2^31 codes and results."""
    rows, inner = 2**20 + 77, 2056
    x = torch.zeros((rows, inner), dtype=torch.bfloat16, device=DEV)
    x[-300:] = torch.randn((300, inner), device=DEV).to(x.dtype)
    w, s = quantize_int8(torch.randn((2056, inner), device=DEV))
    out = linear_int8(x, w, s)
    assert out.numel() > 2**31
    assert_within(out[-300:], *dense_torch.linear_int8(x[-300:], w, s, None, None, None), "out")
    assert not out[:-300].any()
    codes, _ = quantize_int8(x)
    assert torch.equal(codes[-300:], dense_torch.quantize(x[-300:])[0])


def test_refused_on_the_device():
    x, w, s, b, r = make(8, 16, 6, torch.float32)
    for call, error, message in (
            (lambda: linear_int8(x, w.cpu(), s), RuntimeError, "weight must be a ROCm device tensor"),
            (lambda: linear_int8(x, w, s.cpu()), RuntimeError, "weight_scale must be a ROCm"),
            (lambda: linear_int8(x, w, s, b.cpu()), RuntimeError, "bias must be a ROCm"),
            (lambda: linear_int8(x, w.float(), s), TypeError, "weight must be int8"),
            (lambda: linear_int8(x, w, s[:3]), ValueError, "weight_scale must be"),
            (lambda: linear_int8(x, w, s, residual=r[:3]), ValueError, "residual must have"),
            (lambda: linear_int8(x, w, s, activation="silu"), ValueError, "activation must be"),
            (lambda: linear_int8(x.clone().requires_grad_(), w, s), RuntimeError, "no gradients"),
            (lambda: linear_int8(torch.zeros(1, 131088, device=DEV),
                                 torch.zeros((2, 131088), dtype=torch.int8, device=DEV), s[:2]),
             ValueError, "in_features must be at most"),
            (lambda: torch.jit.trace(lambda t: linear_int8(t, w, s), (x,)), RuntimeError,
             "cannot be traced"),
            (lambda: quantize_int8(x.int()), TypeError, "input must be")):
        with pytest.raises(error, match=message):
            call()
    with torch.no_grad():
        assert torch.equal(linear_int8(x.clone().requires_grad_(), w, s), linear_int8(x, w, s))
    codes, scales = quantize_int8(x.clone().requires_grad_())
    assert not codes.requires_grad and not scales.requires_grad


@pytest.mark.parametrize("rows", [1, 300, 9000, 25000])
def test_streams_and_captured_calls(rows):
    """On another stream; captured, two graphs of it replayed in turn on new inputs with eager
    work in between (each has its own workspace)."""
    x, w, s, b, r = make(rows, 96, 80, torch.bfloat16)
    want = linear_int8(x, w, s, b, residual=r)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = linear_int8(x, w, s, b, residual=r)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        source = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_int8(source, w, s, b, residual=r)
        graphs.append((graph, source, out))
    for replay in range(3):
        for graph, source, out in graphs:
            source.copy_(torch.randn(x.shape, device=DEV) + replay)
            graph.replay()
        torch.cuda.synchronize()
        for _, source, out in graphs:
            assert torch.equal(out, linear_int8(source, w, s, b, residual=r))


@pytest.mark.parametrize("size", [(5, 1024, 57344), (128, 1024, 57344), (130, 1024, 57344),
                                  (60000, 1024, 128), (60000, 1024, 136), (60000, 1024, 320)], ids=str)
def test_borders_of_large_tiles(size):
    x, w, s, b, r = make(*size, torch.bfloat16)
    check(x, w, s, b, r, "relu")


def test_more_rows_than_a_launch_of_row_blocks_holds():
    rows = (1 << 30) + 777
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device=DEV)
    x[-500:] = torch.randn((500, 8), device=DEV).to(x.dtype)
    w, s = quantize_int8(torch.randn((3, 8), device=DEV))
    out = linear_int8(x, w, s)
    assert_within(out[-500:], *dense_torch.linear_int8(x[-500:], w, s, None, None, None), "last rows")
    assert not out[:-500].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_pytorch_path_takes_the_same_codes(dtype):
    """Scales are quotients by 127, which a product with its reciprocal would miss by a step."""
    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn((20000, 96), generator=gen, device=DEV)
    x = (x * torch.exp(torch.randn((20000, 1), generator=gen, device=DEV))).to(dtype)
    codes, scales = quantize_int8(x)
    for got, want in ((quantize_int8_pytorch(x), (codes, scales)),
                      (dense_torch.quantize(x), (codes, scales))):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(24600, 80, 96), (24600, 64, 136), (24600, 64, 128), (25001, 100, 200),
                                  (30007, 16, 512), (24577, 240, 40)], ids=str)
def test_short_rows(size, dtype):
    x, w, s, b, r = make(*size, dtype)
    check(x, w, s, b, r, "relu")
    # a weight that starts between 16-byte boundaries
    buffer = torch.zeros(w.numel() + 16, dtype=torch.int8, device=DEV)
    moved = buffer[3:3 + w.numel()].view(w.shape).copy_(w)
    assert torch.equal(linear_int8(x, moved, s, b, residual=r), linear_int8(x, w, s, b, residual=r))
