"""linear on the GPU against float64, at the sizes, layouts and values where it can go wrong."""

import math

import pytest
import torch

from muspace_amd import (
    checkpoint_int8,
    checkpoint_restore,
    get_last_dispatch_report,
    layer_norm,
    linear,
)
from oracle import dense_torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"


def grid(gen, shape, step, limit, dtype):
    """Random values on a grid: sums of products are float32 numbers, so relu's
    side of zero does not depend on the order of a sum."""
    values = torch.randn(shape, generator=gen, device=DEV)
    return (torch.round(values / step) * step).clamp_(-limit, limit).to(dtype)


def make(rows, inner, outer, dtype, *, bias=True, residual=False, seed=0, exact=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if exact:
        x = grid(gen, (rows, inner), 2.0**-3, 4.0, dtype)
        w = grid(gen, (outer, inner), 2.0**-3, 4.0, dtype)
        b = grid(gen, (outer,), 2.0**-6, 1.0, dtype) if bias else None
    else:
        x = torch.randn((rows, inner), generator=gen, device=DEV).to(dtype)
        w = (torch.randn((outer, inner), generator=gen, device=DEV) / math.sqrt(max(inner, 1))).to(dtype)
        b = torch.randn((outer,), generator=gen, device=DEV).to(dtype) if bias else None
    r = torch.randn((rows, outer), generator=gen, device=DEV).to(dtype) if residual else None
    g = torch.randn((rows, outer), generator=gen, device=DEV).to(dtype)
    return x, w, b, r, g


def assert_within(actual, expected, bound, what):
    assert actual.shape == expected.shape, what
    error = (actual.double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((error / bound.clamp_min(1e-300)).max())} of the bound")


def leaves(*tensors):
    return [None if t is None else t.detach().clone().requires_grad_() for t in tensors]


def check(x, w, b, r, g, activation, checkpoint=None):
    xs, ws, bs, rs = leaves(x, w, b, r)
    out = linear(xs, ws, bs, activation=activation, residual=rs, checkpoint=checkpoint)
    assert get_last_dispatch_report().selected_backend == "hip"
    assert out.dtype == x.dtype
    wanted = [t for t in (xs, ws, bs, rs) if t is not None]
    grads = torch.autograd.grad(out, wanted, g)
    kept = dense_torch.checkpoint(x)[2] if checkpoint else None
    results, bounds = dense_torch.linear(x, w, b, activation, r, g, kept)
    if b is None:
        results, bounds = results[:3], bounds[:3]
    got = [out.detach(), *grads[:len(results) - 1]]
    for name, a, e, t in zip(("out", "grad_input", "grad_weight", "grad_bias"), got, results,
                             bounds):
        assert_within(a, e, t, name)
    if r is not None:
        assert torch.equal(grads[-1], g)
    with torch.no_grad():
        again = linear(x, w, b, activation=activation, residual=r)
    assert torch.equal(again, out.detach())  # the same call without a graph


SIZES = [
    (1, 1, 1), (1, 256, 256), (2, 8, 3), (3, 5, 7), (17, 33, 65), (31, 64, 32), (33, 129, 40),
    (130, 256, 520), (300, 96, 64), (257, 203, 131), (1000, 40, 24),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
def test_small_sizes(size, activation, dtype):
    check(*make(*size, dtype, residual=activation != "relu"), activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    ("size", "activation"),
    [((20011, 64, 32), "relu"), ((40000, 96, 160), "relu"), ((33001, 131, 77), "gelu"),
     ((6000, 520, 1030), "relu"), ((2049, 1024, 256), None), ((513, 2048, 300), "gelu")], ids=str)
def test_larger_sizes(size, activation, dtype):
    check(*make(*size, dtype, residual=True), activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(65, 70, 90), (700, 256, 128)], ids=str)
def test_ordinary_values(size, dtype):
    """Values with all their bits (no relu: its side of zero is the sum's)."""
    for activation in (None, "gelu"):
        check(*make(*size, dtype, residual=True, exact=False, seed=3), activation)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_bias_and_residual(dtype):
    check(*make(77, 64, 48, dtype, bias=False), "relu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", [None, "relu"])
@pytest.mark.parametrize("size", [(1, 1, 1), (5, 31, 9), (64, 32, 64), (300, 100, 64),
                                  (20011, 96, 136), (2049, 1000, 256)], ids=str)
def test_checkpoint(size, activation, dtype):
    x, w, b, r, g = make(*size, dtype, residual=True)
    gen = torch.Generator(device=DEV).manual_seed(9)
    # blocks of very different sizes, few of them held exactly by the codes
    scale = torch.exp2(torch.randint(-6, 7, (size[0], 1), generator=gen, device=DEV).float())
    if activation is None:
        x = (torch.randn(size[:2], generator=gen, device=DEV) * scale).to(dtype)
    check(x, w, b, r, g, activation, checkpoint="int8")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 31, 32, 33, 100, 256])
def test_checkpoint_codes_are_exact(cols, dtype):
    gen = torch.Generator(device=DEV).manual_seed(cols)
    info = torch.finfo(dtype)
    x = torch.randn((70, cols), generator=gen, device=DEV)
    x *= torch.exp2(torch.randint(-40, 12, (70, 1), generator=gen, device=DEV).float())
    x = x.to(dtype)
    x[3] = 0.0
    x[4] = info.max
    x[5] = -info.max
    x[6] = info.smallest_normal
    x[7] = info.smallest_normal / 4  # subnormal
    x[8, 0] = math.inf
    x[9, cols - 1] = math.nan
    x[10] = 127.0
    x[11] = 127.5
    x[12] = -63.5
    codes, scales = checkpoint_int8(x)
    e_codes, e_scales, e_values = dense_torch.checkpoint(x)
    assert torch.equal(codes, e_codes)
    assert torch.equal(scales, e_scales)
    restored = checkpoint_restore(codes, scales, cols, dtype)
    assert torch.equal(torch.nan_to_num(restored.double(), nan=-1.0),
                       torch.nan_to_num(e_values, nan=-1.0))
    cpu = checkpoint_int8(x.cpu())
    assert torch.equal(cpu[0], codes.cpu()) and torch.equal(cpu[1], scales.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize(
    ("inner", "outer", "activation"),
    [(3, 5, "relu"), (8, 1, None), (9, 130, "relu"), (203, 611, "gelu"), (512, 64, "relu"),
     (1027, 70, "relu"), (2048, 24, "gelu"), (4112, 33, None)], ids=str)
def test_few_rows(rows, inner, outer, activation, dtype):
    check(*make(rows, inner, outer, dtype, residual=True), activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner", [3, 64, 203, 2051])
def test_few_rows_at_any_address(inner, dtype):
    """The values around each tensor are NaN and must not be read into a result; NaN and
    infinity inside mark their row (x) or column (W) alone."""
    x, w, b, r, g = make(3, inner, 37, dtype, residual=True)

    def shifted(t):
        buffer = torch.full((t.numel() + 9,), math.nan, dtype=t.dtype, device=DEV)
        view = buffer[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    xs, ws, bs, rs = (shifted(t) for t in (x, w, b, r))
    results, bounds = dense_torch.linear(x, w, b, "relu", r, g)
    clean = linear(xs, ws, bs, activation="relu", residual=rs)
    assert_within(clean, results[0], bounds[0], "shifted")
    xs[1, inner - 1] = math.nan
    ws[36, 0] = math.nan
    out = linear(xs, ws, bs, activation="relu", residual=rs)
    assert out[1].isnan().all() and out[:, 36].isnan().all()
    assert torch.equal(out[::2, :36], clean[::2, :36])


def test_one_row_and_most_columns():
    """The most columns that a call takes, every product one value of W: exact."""
    w = torch.arange(1 << 20, device=DEV, dtype=torch.int32).to(torch.float32)[:, None]
    assert torch.equal(linear(torch.full((1, 1), 0.5, device=DEV), w), 0.5 * w.t())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 1, 1), (5, 31, 9), (70, 64, 40), (300, 100, 64),
                                  (9000, 203, 136), (20011, 96, 512), (50001, 200, 260)], ids=str)
def test_checkpoint_of_the_forward_is_the_checkpoint_alone(native_lib, size, dtype):
    """The forward's kernels write the checkpoint as they read the input: the same bytes,
    every one of them, and the same output."""
    rows, inner, outer = size
    x, w, b, _, _ = make(*size, dtype, exact=False)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x *= torch.exp2(torch.randint(-8, 8, (rows, 1), generator=gen, device=DEV).float()).to(dtype)
    x[0] = 0.0
    if rows > 2:
        x[1, inner - 1], x[2, 0] = math.inf, math.nan
    padded = (inner + 31) // 32 * 32
    codes = torch.full((rows + 1, padded), 99, dtype=torch.int8, device=DEV)
    scales = torch.full((rows + 1, padded // 32), 99, dtype=torch.uint8, device=DEV)
    out, plain = (torch.empty((rows, outer), dtype=dtype, device=DEV) for _ in range(2))
    native_lib.linear_forward(x, w, b, None, out, None, 0, codes[:rows], scales[:rows])
    native_lib.linear_forward(x, w, b, None, plain, None, 0)
    assert torch.equal(out.view(torch.uint8), plain.view(torch.uint8))
    want = checkpoint_int8(x)
    assert torch.equal(codes[:rows], want[0]) and torch.equal(scales[:rows], want[1])
    assert codes[rows].eq(99).all() and scales[rows].eq(99).all()  # rows behind: as they were


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype):
    for rows, inner, outer in ((0, 16, 8), (5, 16, 0), (5, 0, 8), (0, 0, 8)):
        x, w, b, r, g = make(rows, inner, outer, dtype, residual=True)
        xs, ws, bs, rs = leaves(x, w, b, r)
        out = linear(xs, ws, bs, activation="relu", residual=rs)
        expected = torch.relu(x.float() @ w.float().t() + b.float()) + r.float()
        torch.testing.assert_close(out.float(), expected, rtol=8e-3, atol=8e-3)
        dx, dw, db, dr = torch.autograd.grad(out, [xs, ws, bs, rs], g)
        dz = g.float() * ((x.float() @ w.float().t() + b.float()) > 0)
        assert torch.equal(dr, g)
        assert dx.shape == x.shape and not dx.any()
        assert dw.shape == w.shape and not dw.any()
        torch.testing.assert_close(db.float(), dz.sum(0), rtol=8e-3, atol=8e-3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(100, 64, 96), (3000, 256, 128)], ids=str)
def test_unaligned_tensors(size, dtype):
    """Sizes of the fast kernels at addresses one value off."""
    x, w, b, r, g = make(*size, dtype, residual=True)

    def shifted(t):
        buffer = torch.full((t.numel() + 9,), math.nan, dtype=t.dtype, device=DEV)
        view = buffer[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    xs, ws, bs, rs, gs = (shifted(t) for t in (x, w, b, r, g))
    for t in (xs, ws, bs, rs):
        t.requires_grad_()
    out = linear(xs, ws, bs, activation="relu", residual=rs)
    grads = torch.autograd.grad(out, [xs, ws, bs], gs)
    results, bounds = dense_torch.linear(x, w, b, "relu", r, g)
    for a, e, t in zip([out.detach(), *grads], results, bounds):
        assert_within(a, e, t, "unaligned")


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_leading_dimensions(dtype):
    x, w, b, r, g = make(6 * 50, 64, 40, dtype, residual=True)
    results, bounds = dense_torch.linear(x, w, b, "relu", r, g)
    xs = x.view(6, 50, 64).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()
    ws = w.t().contiguous().t().requires_grad_()
    bs = torch.stack([b, b], -1)[:, 0].requires_grad_()
    rs = torch.cat([r, r], -1)[:, :40].view(6, 50, 40).requires_grad_()
    gs = torch.cat([g, g], -1)[:, :40].view(6, 50, 40)
    assert not xs.is_contiguous() and not ws.is_contiguous() and not bs.is_contiguous()
    out = linear(xs, ws, bs, activation="relu", residual=rs)
    assert out.shape == (6, 50, 40)
    dx, dw, db = torch.autograd.grad(out, [xs, ws, bs], gs)
    assert dx.shape == xs.shape and dw.shape == ws.shape
    for a, e, t in zip([out.view(-1, 40), dx.reshape(-1, 64), dw, db], results, bounds):
        assert_within(a.detach(), e, t, "strides")


@pytest.mark.parametrize("dtype", DTYPES)
def test_expanded_gradient(dtype):
    """The gradient of a sum is one value seen everywhere (stride 0)."""
    x, w, b, _, _ = make(50, 40, 24, dtype)
    xs, ws, bs = leaves(x, w, b)
    linear(xs, ws, bs).sum().backward()
    results, bounds = dense_torch.linear(x, w, b, None, None, torch.ones_like(x[:, :1]).expand(50, 24))
    for a, e, t in zip([xs.grad, ws.grad, bs.grad], results[1:], bounds[1:]):
        assert_within(a, e, t, "expanded")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(300, 40, 72), (9000, 72, 136), (257, 203, 131)], ids=str)
def test_infinities_and_nan_stay_in_their_rows_and_columns(size, dtype):
    """A row of x with NaN, next to rows whose tail is read in the same step, marks
    its own results only; so does a column of dz."""
    rows, inner, outer = size
    x, w, b, _, g = make(*size, dtype)
    clean = linear(x, w, b)
    x[7] = math.nan
    x[rows - 1, 0] = math.inf
    out = linear(x, w, b)
    assert out[7].isnan().all()
    assert not out[rows - 1].isfinite().logical_and(w[:, 0] != 0).any()
    rest = [i for i in range(rows) if i not in (7, rows - 1)]
    assert torch.equal(out[rest], clean[rest])
    x, w, b, _, g = make(*size, dtype)
    xs, ws, bs = leaves(x, w, b)
    g[5, 3] = math.nan
    dx, dw, db = torch.autograd.grad(linear(xs, ws, bs), [xs, ws, bs], g)
    assert dx[5].isnan().all() and dx[:5].isfinite().all() and dx[6:].isfinite().all()
    assert dw[3].isnan().all() and dw[:3].isfinite().all() and dw[4:].isfinite().all()
    assert db[3].isnan() and db[:3].isfinite().all() and db[4:].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 30000])
def test_gelu_far_from_zero(rows, dtype):
    """Pre-activations past float16's range (kept as infinities there) and infinite ones:
    the limits' values and slopes, not 0 * inf."""
    x = torch.full((rows, 4), 200.0, device=DEV, dtype=dtype)
    w = torch.tensor([[200.0] * 4, [-200.0] * 4, [3.0] * 4, [-3.0] * 4, [0.01] * 4], device=DEV).to(dtype)
    xs, ws = leaves(x, w)
    out = linear(xs, ws, activation="gelu")
    g = torch.ones_like(out)
    dx, dw = torch.autograd.grad(out, [xs, ws], g)
    assert (out[:, 1] == 0).all() and (out[:, 3] == 0).all()
    if dtype != torch.float16:
        assert out.isfinite().all()
    assert dw[1].eq(0).all() and dw[3].eq(0).all() and dx.isfinite().all()
    x[5] = math.inf
    out = linear(x, w, activation="gelu")
    assert (out[5, [0, 2, 4]] == math.inf).all() and (out[5, [1, 3]] == 0).all()
    x[5] = math.nan
    assert linear(x, w, activation="gelu")[5].isnan().all()


def test_float32_keeps_an_absolute_precision():
    """Small float32 values: to 2^-134 each in the product of many rows, exact in few."""
    for rows, step in ((20000, 2.0**-134), (50, 0.0)):
        gen = torch.Generator(device=DEV).manual_seed(2)
        x = torch.randn((rows, 64), generator=gen, device=DEV) * 2.0**-112
        w = torch.randn((512, 64), generator=gen, device=DEV) * 2.0**90
        out = linear(x, w)
        results, bounds = dense_torch.linear(x, w, None, None, None)
        slack = step * w.double().abs().sum(1)
        assert_within(out, results[0], bounds[0] + slack, "small")


@pytest.mark.parametrize("size", [(40, 40, 24), (9000, 72, 136), (257, 203, 131)], ids=str)
def test_float32_over_its_whole_range(size):
    """float32 is multiplied as bfloat16 numbers: values past that type's range (finite in
    float32), infinities and very small values must come out as float32 has them."""
    rows, inner, outer = size
    x, w, b, _, g = make(*size, torch.float32, exact=False, seed=4)
    w = torch.where(w.abs() < 2.0**-6, 2.0**-6, w)
    top = torch.finfo(torch.float32).max
    x[3] = 0.0
    x[3, 5] = top  # rounds to an infinity in bfloat16
    w[:, 5] = w[:, 5].clamp(-0.5, 0.5)
    x[4] *= 2.0**-100
    x[rows - 1, 7] = -math.inf
    check_rows = [i for i in range(rows) if i != rows - 1]
    out = linear(x, w, b)
    results, bounds = dense_torch.linear(x[check_rows], w, b, None, None)
    assert_within(out[check_rows], results[0], bounds[0], "out")
    assert torch.equal(out[rows - 1], torch.where(w[:, 7] > 0, -math.inf, math.inf))
    relu = linear(x, w, b, activation="relu")
    assert torch.equal(relu, torch.relu(out))
    # the same of a gradient: dz^T x and dz W in their tiles
    g[2] = 0.0
    g[2, 3] = top
    xs, ws, bs = leaves(*make(*size, torch.float32, exact=False, seed=8)[:3])
    with torch.no_grad():
        xs[2].clamp_(-0.4, 0.4)
        ws[3].clamp_(-0.4, 0.4)
    grads = torch.autograd.grad(linear(xs, ws, bs), [xs, ws, bs], g)
    results, bounds = dense_torch.linear(xs.detach(), ws.detach(), bs.detach(), None, None, g)
    for a, e, t in zip(grads, results[1:], bounds[1:]):
        assert_within(a, e, t, "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
def test_relu_masks_whatever_the_gradient_holds(dtype):
    """Where relu is off, an infinite or NaN gradient counts as zero; a NaN
    pre-activation passes its gradient on."""
    x, w, b, _, g = make(90, 32, 44, dtype)
    off = (x.double() @ w.double().t() + b.double()) <= 0
    dirty = torch.where(off, torch.tensor(math.nan, device=DEV, dtype=dtype), g)
    xs, ws, bs = leaves(x, w, b)
    out = linear(xs, ws, bs, activation="relu")
    got = torch.autograd.grad(out, [xs, ws, bs], dirty, retain_graph=True)
    want = torch.autograd.grad(out, [xs, ws, bs], g)
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    x[4] = math.nan
    xs, ws, bs = leaves(x, w, b)
    out = linear(xs, ws, bs, activation="relu")
    assert out[4].isnan().all()
    db, = torch.autograd.grad(out, [bs], torch.ones_like(out))
    passed = ~off
    passed[4] = True
    assert torch.equal(db.float(), passed.sum(0).float().to(dtype).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_of_infinities_reads_back_as_nan(dtype):
    x, w, b, _, g = make(40, 70, 16, dtype)
    x[3, 40] = math.inf
    xs, ws, bs = leaves(x, w, b)
    out = linear(xs, ws, bs, checkpoint="int8")
    dx, dw, db = torch.autograd.grad(out, [xs, ws, bs], g)
    assert dw[:, 32:64].isnan().all()  # the block of row 3
    assert dw[:, :32].isfinite().all() and dw[:, 64:].isfinite().all()
    assert dx.isfinite().all() and db.isfinite().all()


def test_single_gradients():
    """Each gradient alone equals the one computed with the others."""
    x, w, b, r, g = make(5000, 96, 72, torch.bfloat16, residual=True)
    xs, ws, bs, rs = leaves(x, w, b, r)
    every = torch.autograd.grad(linear(xs, ws, bs, activation="relu", residual=rs),
                                [xs, ws, bs, rs], g)
    for i in range(4):
        tensors = [t.detach() for t in (x, w, b, r)]
        tensors[i] = tensors[i].clone().requires_grad_()
        out = linear(*tensors[:3], activation="relu", residual=tensors[3])
        alone, = torch.autograd.grad(out, [tensors[i]], g)
        assert torch.equal(alone, every[i])


def test_kept_memory():
    """relu keeps a bit per value, the 8-bit checkpoint 33/32 bytes per input value."""
    rows, inner, outer = 1 << 15, 256, 512
    x, w, b, _, _ = make(rows, inner, outer, torch.bfloat16)
    ws, bs = leaves(w, b)
    before = torch.cuda.memory_allocated()
    out = linear(x.clone(), ws, bs, activation="relu", checkpoint="int8")
    held = torch.cuda.memory_allocated() - before - out.numel() * 2
    assert held <= rows * inner * 33 // 32 + rows * outer // 8 + 4096


def test_large_offsets():
    """More than 2^31 values in the output: 64-bit row offsets."""
    rows, inner, outer = 2**18 + 37, 32, 8200
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = grid(gen, (rows, inner), 2.0**-3, 4.0, torch.bfloat16)
    w = grid(gen, (outer, inner), 2.0**-3, 4.0, torch.bfloat16)
    assert rows * outer > 2**31
    out = linear(x, w, activation="relu")
    for part in (slice(0, 64), slice(rows - 70, rows)):
        results, bounds = dense_torch.linear(x[part], w, None, "relu", None)
        assert_within(out[part], results[0], bounds[0], "large")


def test_repeated_calls_are_bitwise_equal():
    x, w, b, r, g = make(30000, 200, 136, torch.float32, residual=True, exact=False)

    def step():
        xs, ws, bs = leaves(x, w, b)
        out = linear(xs, ws, bs, activation="gelu", residual=r)
        return [out.detach(), *torch.autograd.grad(out, [xs, ws, bs], g)]

    first = step()
    for _ in range(3):
        for a, e in zip(step(), first):
            assert torch.equal(a, e)


def test_side_stream():
    x, w, b, r, g = make(4000, 128, 256, torch.bfloat16, residual=True)
    xs, ws, bs = leaves(x, w, b)
    want_out = linear(xs, ws, bs, activation="relu", residual=r)
    want = torch.autograd.grad(want_out, [xs, ws, bs], g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = linear(xs, ws, bs, activation="relu", residual=r)
        got = torch.autograd.grad(out, [xs, ws, bs], g)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, want_out)
    for a, e in zip(got, want):
        assert torch.equal(a, e)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_captured_step_replays(checkpoint):
    """A layer's block captured with its gradients: every replay, with other work in
    between, equals the eager step on the same inputs."""
    dtype = torch.bfloat16
    x, w1, b1, _, _ = make(5000, 96, 160, dtype, seed=1, exact=False)
    _, w2, b2, _, g = make(5000, 160, 96, dtype, seed=2, exact=False)
    gamma = torch.linspace(0.5, 1.5, 96, device=DEV).to(dtype)
    beta = torch.linspace(-1.0, 1.0, 96, device=DEV).to(dtype)
    params = leaves(x, w1, b1, w2, b2, gamma, beta)

    def step():
        xs, p1, q1, p2, q2, ga, be = params
        hidden = linear(xs, p1, q1, activation="relu", checkpoint=checkpoint)
        y = linear(hidden, p2, q2, residual=xs, checkpoint=checkpoint)
        out = layer_norm(y, ga, be)
        return [out.detach(), *torch.autograd.grad(out, params, g)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        with torch.no_grad():
            params[0].copy_(torch.randn(x.shape, device=DEV) + replay)
            g.copy_(torch.randn(g.shape, device=DEV))
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        for a, e in zip(got, step()):
            assert torch.equal(a, e)


def test_two_graphs_share_a_pool():
    """Two captured steps in one memory pool, replayed in turn: each has its own workspace
    while it runs."""
    x, w, b, _, g = make(20000, 96, 128, torch.bfloat16, seed=1)
    y, v, c, _, h = make(20000, 128, 64, torch.bfloat16, seed=2)
    sets = [(leaves(x, w, b), g), (leaves(y, v, c), h)]

    def step(params, grad):
        out = linear(*params, activation="relu", checkpoint="int8")
        return [out.detach(), *torch.autograd.grad(out, params, grad)]

    want = [step(*s) for s in sets]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for s in sets:
            step(*s)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graphs, results, pool = [], [], None
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            results.append(step(*s))
        pool = graph.pool()
        graphs.append(graph)
    for _ in range(3):
        for graph, result, expected in zip(graphs, results, want):
            graph.replay()
            got = [t.clone() for t in result]
            torch.cuda.synchronize()
            for a, e in zip(got, expected):
                assert torch.equal(a, e)
            step(*sets[0])


def test_streams_at_once():
    """Calls in flight on two streams do not share scratch."""
    x, w, b, _, g = make(60000, 128, 128, torch.bfloat16, seed=1)
    xs, ws, bs = leaves(x, w, b)

    def step():
        return torch.autograd.grad(linear(xs, ws, bs, activation="gelu"), [xs, ws, bs], g)

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(step())
    torch.cuda.synchronize()
    for grads in got:
        for a, e in zip(grads, want):
            assert torch.equal(a, e)


def test_gradients_against_differences():
    """d loss along a random direction of every input, float32, against central differences
    of the float64 formula."""
    x, w, b, r, g = make(60, 48, 36, torch.float32, residual=True, exact=False, seed=5)
    xs, ws, bs, rs = leaves(x, w, b, r)
    grads = torch.autograd.grad(linear(xs, ws, bs, activation="gelu", residual=rs),
                                [xs, ws, bs, rs], g)
    gen = torch.Generator(device=DEV).manual_seed(6)
    h = 1e-4
    for i, grad in enumerate(grads):
        tensors = [t.double() for t in (x, w, b, r)]
        d = torch.randn(tensors[i].shape, generator=gen, device=DEV, dtype=torch.float64)

        def loss(sign):
            moved = list(tensors)
            moved[i] = moved[i] + sign * h * d
            y = dense_torch.gelu(moved[0] @ moved[1].t() + moved[2]) + moved[3]
            return (y * g.double()).sum()

        difference = (loss(1) - loss(-1)) / (2 * h)
        # differences err by h^2 times a third derivative, far below; the gradient by
        # float32 sums of at most 60 * 36 terms along d
        slack = 2160 * dense_torch.SUM_STEP * float((grad.double().abs() * d.abs()).sum()) + 1e-5
        assert abs(float((grad.double() * d).sum() - difference)) <= slack


def test_refused_on_the_device():
    x, w, b, r, g = make(8, 16, 12, torch.float32, residual=True)
    with pytest.raises(RuntimeError, match="weight is on cpu|must be a ROCm device tensor"):
        linear(x, w.cpu(), b)
    with pytest.raises(RuntimeError, match="residual must be a ROCm device tensor"):
        linear(x, w, b, residual=r.cpu())
    for change, error, message in (
            ({"input": x.double()}, TypeError, "input must be"),
            ({"input": x[0, 0]}, ValueError, "at least one dimension"),
            ({"weight": w[:, :8]}, ValueError, "weight must be"),
            ({"weight": w[0]}, ValueError, "weight must be"),
            ({"weight": w.half()}, TypeError, "weight must be"),
            ({"bias": b[:3]}, ValueError, "bias must be"),
            ({"bias": b.half()}, TypeError, "bias must be"),
            ({"residual": r[:1]}, ValueError, "residual must have"),
            ({"residual": r.view(2, 4, 12)}, ValueError, "residual must have"),
            ({"residual": r.half()}, TypeError, "residual must be"),
            ({"activation": "silu"}, ValueError, "activation must be"),
            ({"checkpoint": "fp8"}, ValueError, "checkpoint must be"),
            ({"backend": "cuda"}, RuntimeError, "unknown backend")):
        args = {"input": x, "weight": w, "bias": b, "residual": r, **change}
        with pytest.raises(error, match=message):
            linear(args.pop("input"), args.pop("weight"), args.pop("bias"), **args)
    assert torch.equal(linear(x, w, b, backend="hip"), linear(x, w, b))
    reference = linear(x, w, b, backend="reference")
    assert get_last_dispatch_report().selected_backend == "reference"
    torch.testing.assert_close(reference, linear(x, w, b), rtol=1e-5, atol=1e-5)
    xs = x.clone().requires_grad_()
    grad, = torch.autograd.grad(linear(xs, w, b), [xs], g)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(linear(xs, w, b), [xs], g, create_graph=True)[0].sum().backward()


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("activation", [0, 1, 2])
def test_tensor_level_entries(native_lib, activation, checkpoint):
    """The library's checked entries on caller-owned tensors give the operator's results."""
    x, w, b, r, g = make(700, 96, 72, torch.bfloat16, residual=True)
    name = {0: None, 1: "relu", 2: "gelu"}[activation]
    xs, ws, bs = leaves(x, w, b)
    want_out = linear(xs, ws, bs, activation=name, residual=r,
                      checkpoint="int8" if checkpoint else None)
    want = torch.autograd.grad(want_out, [xs, ws, bs], g)
    kept = {0: None, 1: torch.empty((2, 700, 8), dtype=torch.uint8, device=DEV),
            2: torch.empty((700, 72), dtype=torch.bfloat16, device=DEV)}[activation]
    out = torch.empty((700, 72), dtype=torch.bfloat16, device=DEV)
    codes = scales = None
    if checkpoint:
        codes = torch.empty((700, 96), dtype=torch.int8, device=DEV)
        scales = torch.empty((700, 3), dtype=torch.uint8, device=DEV)
    native_lib.linear_forward(x, w, b, r, out, kept, activation, codes, scales)
    assert torch.equal(out, want_out)
    got = [torch.full_like(t, math.nan) for t in (x, w, b)]
    native_lib.linear_backward(g, None if checkpoint else x, codes, scales, w, kept, *got,
                               (72, 96), activation)
    for a, e in zip(got, want):
        assert torch.equal(a, e)


def test_tensor_level_entries_refuse(native_lib):
    x, w, b, r, g = make(8, 16, 12, torch.float16, residual=True)
    out = torch.empty_like(r)
    good = dict(input=x, weight=w, bias=b, residual=r, output=out, kept=None, activation=0)
    for change, message in (
            ({"weight": w[:, :8]}, "contiguous"),
            ({"weight": w.float()}, "weight must be float16"),
            ({"weight": w.cpu()}, "ROCm device tensor"),
            ({"bias": b[:5].contiguous()}, "bias must have shape"),
            ({"output": out[:4]}, "output must have shape"),
            ({"kept": out, "activation": 1}, "relu_mask must be uint8"),
            ({"kept": out[:3], "activation": 2}, "pre_activation must have shape"),
            ({"kept": out}, "nothing is kept")):
        with pytest.raises(RuntimeError, match=message):
            native_lib.linear_forward(**{**good, **change})
    with pytest.raises(RuntimeError, match="codes must have shape"):
        native_lib.linear_checkpoint(x, torch.empty((8, 16), dtype=torch.int8, device=DEV),
                                     torch.empty((8, 1), dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="null tensor pointer"):  # neither input nor codes
        native_lib.linear_backward(g, None, None, None, w, None, torch.empty_like(x),
                                   torch.empty_like(w), None, (12, 16), 0)
