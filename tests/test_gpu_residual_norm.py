"""dropout and residual_norm on the GPU against float64."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from muspace_amd import dropout, get_last_dispatch_report, residual_norm
from muspace_amd.ops.residual_norm import residual_norm_pytorch
from oracle import block_torch, dense_torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"
VECTORS = ("weight", "bias", "gate", "post_weight", "post_bias")


def mask(shape, p, seed, offset):
    """The generator's definition on the device (integers of 64 bits; tied to the
    oracle's by test_masks)."""
    from muspace_amd.ops.dropout import kept_elements

    return kept_elements(shape, p, seed, offset, DEV)


def assert_within(actual, expected, bound, what):
    assert actual.shape == expected.shape, what
    error = (actual.double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((error / bound.clamp_min(1e-300)).max())} of the bound")


# ------------------------------------------------------------------ dropout ---


@pytest.mark.parametrize("seed", [0, 2**31, 2**64 - 1])
@pytest.mark.parametrize("offset", [0, 2**32 + 5, 2**64 - 1])
def test_masks(seed, offset):
    out = dropout(torch.ones(1003, device=DEV), 0.37, seed=seed, offset=offset)
    assert get_last_dispatch_report().selected_backend == "hip"
    want = block_torch.kept(0, 1003, 0.37, seed, offset)
    assert torch.equal((out != 0).cpu(), want)
    assert torch.equal(mask((1003,), 0.37, seed, offset).cpu(), want)
    if seed < 2**63:
        tensor = torch.tensor([seed], device=DEV)
        assert torch.equal(dropout(torch.ones(1003, device=DEV), 0.37, seed=tensor, offset=offset), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("count", [1, 3, 4, 7, 8, 9, 63, 1001, 4096, 70001, 3000017])
def test_dropout_sizes(count, residual, dtype):
    gen = torch.Generator(device=DEV).manual_seed(count)
    x, r, g = (torch.randn(count, generator=gen, device=DEV).to(dtype) for _ in range(3))
    xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
    out = dropout(xs, 0.3, seed=9, offset=4, residual=rs if residual else None)
    keep = mask((count,), 0.3, 9, 4)
    assert_within(out.detach(), *block_torch.dropout(x, keep, 0.3, r if residual else None), "out")
    grads = torch.autograd.grad(out, [xs, rs] if residual else [xs], g)
    assert_within(grads[0], *block_torch.dropout(g, keep, 0.3), "grad")
    assert not residual or torch.equal(grads[1], g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [0.0, 1e-11, 1 - 2.0**-33, 1.0])
def test_dropout_at_the_ends(p, dtype):
    x = torch.randn((5, 77), device=DEV).to(dtype)
    x[0, 0], x[1, 1] = math.inf, math.nan
    out = dropout(x, p, seed=1)
    if p < 0.5:
        assert torch.equal(out[2:], x[2:]) and out[0, 0] == math.inf and out[1, 1].isnan()
    else:  # what is dropped is zero, whatever it was
        assert not out.any()


def test_dropout_views_alignment_and_far_elements():
    x = torch.randn((60, 50), device=DEV).bfloat16()
    want = dropout(x, 0.4, seed=2)
    assert torch.equal(dropout(x.t().contiguous().t(), 0.4, seed=2), want)
    buffer = torch.zeros(3001, dtype=torch.bfloat16, device=DEV)
    buffer[1:].copy_(x.view(-1))
    assert torch.equal(dropout(buffer[1:].view(60, 50), 0.4, seed=2, residual=buffer[1:].view(60, 50)),
                       dropout(x, 0.4, seed=2, residual=x))
    assert torch.equal(dropout(torch._neg_view(x), 0.4, seed=2), -want)
    # elements past 2^32
    n = 2**32 + 1009
    ones = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    out = dropout(ones, 0.5, seed=3)
    for first in (0, 2**31 - 500, 2**32 - 500):
        assert torch.equal((out[first:first + 1000] != 0).cpu(), block_torch.kept(first, 1000, 0.5, 3, 0))
    del ones, out


def test_dropout_seed_tensor_changed_before_the_backward_is_refused():
    x = torch.randn(100, device=DEV, requires_grad=True)
    seed = torch.tensor([5], device=DEV)
    out = dropout(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ------------------------------------------------------------ residual norm ---


def make(rows, cols, dtype, names=VECTORS, wdtype=None, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    t = {"block": normal(rows, cols).to(dtype),
         "residual": (normal(rows, cols) * torch.exp(0.5 * normal(cols)) + 0.5 * normal(cols)).to(dtype)}
    for name in names:
        centre = 0.0 if name.endswith("bias") else 1.0
        t[name] = (centre + 0.3 * normal(cols)).to(wdtype or dtype)
    return t, normal(rows, cols).to(dtype), normal(rows, cols).to(dtype)


def check(t, g, gs, p=0.0, **kwargs):
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    normed, stream = residual_norm(**leaves, dropout_p=p, seed=7, offset=1, **kwargs)
    assert get_last_dispatch_report().selected_backend == "hip"
    keep = mask(t["block"].shape, p, 7, 1) if p else None
    want = block_torch.residual_norm(**t, p=p, keep=keep, grad=g, grad_stream=gs, **kwargs)
    outs = [o for o, d in ((normed, g), (stream, gs)) if d is not None]
    grads = torch.autograd.grad(outs, list(leaves.values()), [d for d in (g, gs) if d is not None],
                                allow_unused=g is None)
    got = {"normed": normed.detach(), "stream": stream.detach(), **dict(zip(leaves, grads))}
    for name, (value, bound) in want.items():
        assert_within(got[name], value, bound, name)
        if name in leaves:
            assert got[name].dtype == t[name].dtype
    with torch.no_grad():
        again = residual_norm(**t, dropout_p=p, seed=7, offset=1, **kwargs)
        assert torch.equal(again[0], normed) and torch.equal(again[1], stream)
        assert torch.equal(residual_norm(**t, dropout_p=p, seed=7, offset=1, return_stream=False,
                                         **kwargs), normed)
    return got


SIZES = [(1, 1), (1, 2), (3, 7), (5, 64), (33, 128), (64, 129), (300, 256), (77, 255), (1, 512),
         (130, 513), (41, 1024), (19, 1500), (12, 2048), (9, 2051), (5, 4096), (4, 4100), (3, 9000),
         (2, 16400), (2, 40001), (20000, 96), (40013, 256), (9001, 611)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "cols"), SIZES)
def test_sizes(rows, cols, dtype):
    """Rows of every number of lanes, the everyday call and the one with everything."""
    t, g, gs = make(rows, cols, dtype)
    check({k: t[k] for k in ("block", "residual", "weight", "bias")}, g, gs, p=0.1)
    check(t, g, gs, p=0.3, norm="rms", post_norm="layer", residual_scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("cols", [96, 1000, 5000])
def test_kinds(cols, post, norm, dtype):
    t, g, gs = make(60, cols, dtype)
    if post is None:
        t = {k: v for k, v in t.items() if not k.startswith("post")}
    for p in (0.0, 0.25):
        check(t, g, gs, p=p, norm=norm, post_norm=post, residual_scale=1.5)
    check({k: t[k] for k in ("block", "residual")}, g, gs, norm=norm, post_norm=post)
    check({k: t[k] for k in ("block", "residual", "gate")}, g, gs, norm=norm, post_norm=post)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [40, 203, 1024, 9000])
def test_float32_vectors_of_a_16_bit_block(cols, dtype):
    t, g, gs = make(70, cols, dtype, wdtype=torch.float32)
    check(t, g, gs, p=0.2, post_norm="rms")


@pytest.mark.parametrize("cols", [256, 5000])
def test_gradients_of_one_output(cols):
    t, g, gs = make(90, cols, torch.float32)
    check(t, g, None, p=0.2, post_norm="layer")
    got = check(t, None, gs, p=0.2, post_norm="layer")
    assert got["weight"] is None and got["bias"] is None
    plain = {k: t[k] for k in ("block", "residual")}
    got = check(plain, None, gs)
    assert torch.equal(got["block"], gs) and torch.equal(got["residual"], gs)


def test_one_tensor_as_block_and_residual():
    """Gradients of both add up, and gradients that are one result are not one tensor."""
    t, g, gs = make(60, 256, torch.float32, names=("weight", "bias"))
    for kwargs in ({}, {"dropout_p": 0.3, "seed": 2}, {"residual_scale": 0.5}):
        a, b = (t["block"].clone().requires_grad_() for _ in range(2))
        torch.autograd.backward(residual_norm(a, b, t["weight"], t["bias"], **kwargs), [g, gs])
        x = t["block"].clone().requires_grad_()
        torch.autograd.backward(residual_norm(x, x, t["weight"], t["bias"], **kwargs), [g, gs])
        assert torch.equal(x.grad, a.grad + b.grad)
        kept = b.grad.clone()
        a.grad.zero_()
        assert torch.equal(b.grad, kept)


@pytest.mark.parametrize("scale", [1e300, -math.inf])
def test_residual_scale_is_a_float32_number(scale):
    t, _, _ = make(4, 8, torch.float32, names=())
    with pytest.raises(ValueError, match="residual_scale must be a finite float32"):
        residual_norm(**t, residual_scale=scale)


def test_single_gradients_and_repeats():
    t, g, gs = make(9000, 200, torch.bfloat16)

    def grads(names):
        leaves = {k: v.clone().requires_grad_(k in names) for k, v in t.items()}
        outs = residual_norm(**leaves, post_norm="layer", dropout_p=0.1, seed=3)
        return torch.autograd.grad(outs, [leaves[k] for k in names], [g, gs])

    every = dict(zip(t, grads(list(t))))
    for a, e in zip(grads(list(t)), every.values()):
        assert torch.equal(a, e)
    for name in t:
        assert torch.equal(grads([name])[0], every[name]), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 1024, 1500])
def test_rows_far_from_zero_and_constant_rows(cols, dtype):
    """The norm is of the sum before it is rounded: a 16-bit stream at 100 loses what the norm
    of the sum keeps."""
    t, g, gs = make(64, cols, dtype, names=("weight", "bias"))
    t["residual"][:32] = 100.0
    t["block"][:32] = t["block"][:32] * 0.02
    t["residual"][40], t["block"][40] = 3.5, 0.25
    assert torch.equal(residual_norm(**t)[0][40], t["bias"])
    keep = [i for i in range(64) if i != 40]  # (without a spread: s is 1 / sqrt(eps))
    check({k: v[keep] if v.dim() == 2 else v for k, v in t.items()}, g[keep], gs[keep])
    other, stream = residual_norm(**t)
    if dtype == torch.float32:  # the stream is the sum
        results, bounds = dense_torch.layer_norm(stream, t["weight"], t["bias"], 1e-5)
        assert_within(other, results[0], 2 * bounds[0], "normed")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("post", [None, "rms"])
def test_precision(post, dtype):
    """Root mean squares: every result errs by its own rounding alone (2% of room for float32)."""
    names = ("weight", "bias", "gate", "post_weight") if post else ("weight", "bias")
    t, g, gs = make(6000, 512, dtype, names=names)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    outs = residual_norm(**leaves, post_norm=post, dropout_p=0.1, seed=7)
    grads = torch.autograd.grad(outs, list(leaves.values()), [g, gs])
    want = block_torch.residual_norm(**t, post_norm=post, p=0.1, keep=mask((6000, 512), 0.1, 7, 0),
                                     grad=g, grad_stream=gs)

    def rms(a, e):
        return float((a.double() - e).square().mean().sqrt())

    for name, a in {"normed": outs[0], "stream": outs[1], **dict(zip(leaves, grads))}.items():
        e = want[name][0]
        assert rms(a, e) <= 1.02 * rms(e.to(dtype), e), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 5000])
def test_infinity_and_nan_stay_in_their_rows(cols, dtype):
    t, g, gs = make(50, cols, dtype)
    kwargs = {"post_norm": "rms", "dropout_p": 0.5, "seed": 1}
    clean = residual_norm(**t, **kwargs)
    t["block"][7, 5], t["residual"][8, 255], t["residual"][9, 0] = math.nan, math.inf, -math.inf
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    outs = residual_norm(**leaves, **kwargs)
    rest = [i for i in range(50) if i not in (7, 8, 9)]
    for a, e in zip(outs, clean):
        assert torch.equal(a[rest], e[rest])
    assert outs[0][[7, 8, 9]].isnan().all()
    db, dr = torch.autograd.grad(outs, [leaves["block"], leaves["residual"]], [g, gs])
    assert db[rest].isfinite().all() and dr[rest].isfinite().all()
    # without a norm on it, a dropped NaN of the block is gone
    keep = mask((50, cols), 0.5, 1, 0)
    x = torch.zeros_like(t["block"])
    row, col = (~keep).nonzero()[0].tolist()
    x[row, col] = math.nan
    stream = residual_norm(x, torch.ones_like(x), gate=t["gate"], dropout_p=0.5, seed=1)[1]
    assert torch.equal(stream, torch.ones_like(x))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype):
    for shape in ((0, 64), (3, 0), (2, 0, 5), (0, 20000)):
        x, w = (torch.ones(s, dtype=dtype, device=DEV, requires_grad=True) for s in (shape, shape[-1:]))
        normed, stream = residual_norm(x, x, w, gate=w, dropout_p=0.5, seed=1)
        assert normed.shape == stream.shape == shape
        dx, dw = torch.autograd.grad([normed, stream], [x, w], [normed, stream])
        assert dx.shape == shape and not dw.any()
        assert dropout(x, 0.5, seed=1).shape == shape


@pytest.mark.parametrize("cols", [256, 100])
def test_unaligned_strided_and_negated(cols):
    t, g, gs = make(120, cols, torch.float16)
    kwargs = {"post_norm": "layer", "dropout_p": 0.2, "seed": 5}

    def step(tensors, grads):
        leaves = {k: v.requires_grad_() for k, v in tensors.items()}
        outs = residual_norm(**leaves, **kwargs)
        return [*outs, *torch.autograd.grad(outs, list(leaves.values()), grads)]

    def shifted(v):
        buffer = torch.full((v.numel() + 9,), math.nan, dtype=v.dtype, device=DEV)
        view = buffer[1:1 + v.numel()].view(v.shape)
        view.copy_(v)
        return view

    want = step({k: v.clone() for k, v in t.items()}, [g, gs])
    strided = {k: torch.stack([v, v], -1)[..., 0] for k, v in t.items()}
    negated = {k: torch._neg_view(-v) for k, v in t.items()}
    for got in (step({k: shifted(v) for k, v in t.items()}, [shifted(g), shifted(gs)]),
                step(strided, [g.t().contiguous().t(), gs]),
                step(negated, [torch._neg_view(-g), gs])):
        for a, e in zip(got, want):
            assert torch.equal(a, e)
    shaped = {k: v.view(2, 60, cols) if v.dim() == 2 else v for k, v in t.items()}
    assert torch.equal(residual_norm(**shaped, **kwargs)[0].view(120, cols), want[0])
    one = {k: v[3] if v.dim() == 2 else v for k, v in t.items()}
    normed, _ = residual_norm(**one, post_norm="layer")
    assert normed.shape == (cols,)


def test_large_offsets():
    """More than 2^31 values: 64-bit row offsets and dropout indices."""
    rows, cols = 2**20 + 5, 2056
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2**31
    x[-40:] = torch.randn((40, cols), device=DEV).to(x.dtype)
    normed, stream = residual_norm(x, x, dropout_p=0.5, seed=6)
    keep = block_torch.kept((rows - 2) * cols, 2 * cols, 0.5, 6, 0).view(2, cols).to(DEV)
    want = block_torch.residual_norm(x[-2:], x[-2:], p=0.5, keep=keep)
    assert_within(stream[-2:], *want["stream"], "stream")
    assert_within(normed[-2:], *want["normed"], "normed")


def test_gradients_against_differences():
    t, g, gs = make(30, 72, torch.float32, seed=2)
    kwargs = {"norm": "layer", "post_norm": "rms", "residual_scale": 0.8}
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    outs = residual_norm(**leaves, dropout_p=0.3, seed=2, **kwargs)
    grads = torch.autograd.grad(outs, list(leaves.values()), [g, gs])
    keep = mask((30, 72), 0.3, 2, 0)
    gen = torch.Generator(device=DEV).manual_seed(3)
    step = 1e-4
    for name, grad in zip(leaves, grads):
        d = torch.randn(t[name].shape, generator=gen, device=DEV, dtype=torch.float64)

        def loss(sign):
            moved = {k: v.double() for k, v in t.items()}
            moved[name] = moved[name] + sign * step * d
            out = block_torch.residual_norm(**moved, p=0.3, keep=keep, **kwargs)
            return (out["normed"][0] * g.double()).sum() + (out["stream"][0] * gs.double()).sum()

        difference = (loss(1) - loss(-1)) / (2 * step)
        # float32 sums of at most 72 or 30 terms, of magnitudes up to a few times the
        # gradient's own; differences err by step^2 times a third derivative
        slack = 400 * 2.0**-23 * float((grad.double().abs() * d.abs()).sum()) + 1e-4
        assert abs(float((grad.double() * d).sum() - difference)) <= slack, name


def test_refused_on_the_device():
    t, _, _ = make(8, 16, torch.float32)
    x, r = t["block"], t["residual"]
    for call, error, message in (
            (lambda: residual_norm(x, r.cpu()), RuntimeError, "residual must be a ROCm device tensor"),
            (lambda: residual_norm(x, r, gate=t["gate"].cpu()), RuntimeError, "gate must be a ROCm"),
            (lambda: residual_norm(x, r, dropout_p=0.5, seed=torch.tensor([1])), RuntimeError, "seed must be"),
            (lambda: residual_norm(x.double(), r), TypeError, "block must be"),
            (lambda: residual_norm(x, r[:4]), ValueError, "residual must have"),
            (lambda: residual_norm(x, r, post_weight=t["gate"]), ValueError, "without a post_norm"),
            (lambda: residual_norm(x, r, gate=t["gate"][:3]), ValueError, "gate must be"),
            (lambda: residual_norm(x, r, t["weight"], t["bias"].half()), TypeError, "must be"),
            (lambda: residual_norm(x, r, norm="none"), ValueError, "norm must be"),
            (lambda: dropout(x, 0.5, seed=torch.tensor([1])), RuntimeError, "seed must be"),
            (lambda: dropout(x, 0.5, seed=1, residual=r.cpu()), RuntimeError, "residual must be"),
            (lambda: dropout(x.int(), 0.5, seed=1), TypeError, "input must be"),
            (lambda: dropout(x, 0.5, seed=torch.ones(1, device=DEV)), TypeError, "seed tensor"),
            (lambda: dropout(x, 0.5, seed=1, backend="none"), RuntimeError, "unknown backend")):
        with pytest.raises(error, match=message):
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t["weight"], torch.ones_like(t["weight"]))
        with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
            residual_norm(x, r, dual)
        with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
            dropout(x, 0.5, seed=1, residual=forward_ad.make_dual(r, r))
    with pytest.raises(RuntimeError, match="HIP kernels cannot be traced"):
        torch.jit.trace(lambda v: residual_norm(v, r)[0], (x,))
    xs = x.clone().requires_grad_()
    for out in (dropout(xs, 0.5, seed=1), residual_norm(xs, r)[0]):
        first, = torch.autograd.grad(out.square().sum(), [xs], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate .* twice"):
            first.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_reference_backend_draws_the_same_masks(dtype):
    t, _, _ = make(50, 203, dtype)
    kwargs = {"post_norm": "rms", "dropout_p": 0.5, "seed": 8, "offset": 3}
    a, b = residual_norm(**t, **kwargs), residual_norm(**t, backend="reference", **kwargs)
    keep = mask((50, 203), 0.5, 8, 3)
    want = block_torch.residual_norm(**t, post_norm="rms", p=0.5, keep=keep)
    assert_within(a[1], *want["stream"], "stream")
    assert_within(b[1], *want["stream"], "stream")
    x = t["block"]
    assert torch.equal(dropout(x, 0.5, seed=8), dropout(x, 0.5, seed=8, backend="reference"))
    with torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(residual_norm_pytorch(**t, **kwargs)[0], b[0])


def test_recomputed_blocks():
    """Under torch.utils.checkpoint the second forward draws the first one's masks."""
    from torch.utils.checkpoint import checkpoint

    t, g, gs = make(500, 96, torch.bfloat16)

    def function(block, residual, weight):
        x = dropout(block, 0.2, seed=4, offset=0)
        return residual_norm(x, residual, weight, dropout_p=0.1, seed=4, offset=1)

    def step(call):
        leaves = [t[k].clone().requires_grad_() for k in ("block", "residual", "weight")]
        outs = call(*leaves)
        return [*outs, *torch.autograd.grad(outs, leaves, [g, gs])]

    want = step(function)
    with torch.autograd.graph.save_on_cpu():
        offloaded = step(function)
    for got in (step(lambda *a: checkpoint(function, *a, use_reentrant=False)), offloaded):
        for a, e in zip(got, want):
            assert torch.equal(a, e)


def test_streams_and_captured_steps():
    """On another stream; captured, and replayed with new tensors and a new seed while eager
    work runs in between."""
    t, g, gs = make(9000, 256, torch.bfloat16)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    seed = torch.tensor([11], device=DEV)

    def step(seed=seed):
        x = dropout(leaves["block"], 0.1, seed=seed, offset=0, residual=leaves["residual"])
        outs = residual_norm(**{**leaves, "block": x}, post_norm="rms", dropout_p=0.2, seed=seed,
                             offset=1)
        return [*(o.detach() for o in outs),
                *torch.autograd.grad(outs, list(leaves.values()), [g, gs])]

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
    before = None
    for replay in range(4):
        with torch.no_grad():
            leaves["residual"].copy_(torch.randn(g.shape, device=DEV) + replay)
        seed.add_(1)
        graph.replay()
        got = [v.clone() for v in captured]
        torch.cuda.synchronize()
        for a, e in zip(got, step(11 + replay + 1)):
            assert torch.equal(a, e)
        assert before is None or not torch.equal(before, got[0])
        before = got[0]
