"""Ways to call the dense operators on the GPU besides the plain ones: traced, with
forward-mode derivatives, and of tensors in unusual states."""

import importlib
import math
from contextlib import nullcontext

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import checkpoint_int8, checkpoint_restore, layer_norm, linear

linear_module = importlib.import_module("muspace_amd.ops.linear")  # (the package has the function)

pytestmark = pytest.mark.gpu

DEV = "cuda"


def calls():
    gen = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn((4, 8), generator=gen, device=DEV)
    b = torch.randn(8, generator=gen, device=DEV)
    return {"linear": lambda x: linear(x, w, activation="gelu"),
            "checkpointed": lambda x: linear(x, w, checkpoint="int8"),
            "layer_norm": lambda x: layer_norm(x, b, b)}


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("which", ["linear", "checkpointed", "layer_norm"])
def test_tracing_and_forward_mode_are_refused(which, graph):
    call = calls()[which]
    x = torch.randn((3, 8), device=DEV, requires_grad=graph)
    for trace in (lambda: torch.jit.trace(call, (x,)), lambda: make_fx(call)(x.detach())):
        with pytest.raises(RuntimeError, match="HIP kernels cannot be traced"):
            trace()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
            call(dual)
    # a tensor without a tangent, and where forward mode is off
    assert call(x).isfinite().all()
    with pytest.raises(RuntimeError, match="HIP kernels cannot be traced"):
        torch.jit.trace(lambda t: checkpoint_int8(t)[0], (x.detach(),))


def test_a_weight_with_a_tangent_is_refused():
    x, w = torch.randn((3, 8), device=DEV), torch.randn((4, 8), device=DEV)
    b, r = torch.randn(4, device=DEV), torch.randn((3, 4), device=DEV)
    with forward_ad.dual_level():
        for i in range(1, 4):
            given = [x, w, b, r]
            given[i] = forward_ad.make_dual(given[i], torch.ones_like(given[i]))
            with pytest.raises(RuntimeError, match="linear: the HIP path has no forward-mode"):
                linear(*given[:3], residual=given[3])
        scale = torch.ones(8, device=DEV)
        with pytest.raises(RuntimeError, match="layer_norm: the HIP path has no forward-mode"):
            layer_norm(x, scale, forward_ad.make_dual(scale, scale))


def test_the_reference_backend_is_traced_on_the_device():
    x, w = torch.randn((3, 8), device=DEV), torch.randn((4, 8), device=DEV)
    traced = torch.jit.trace(lambda t: linear(t, w, backend="reference"), (x,))
    y = torch.randn((3, 8), device=DEV)
    torch.testing.assert_close(traced(y), linear(y, w, backend="reference"))


@pytest.mark.parametrize("shape", [(1, 1), (5, 8)])
def test_views_read_with_their_sign_changed(shape):
    """A contiguous view of another tensor's negative (of one value: the imaginary part of a
    conjugate) counts with its own values, as an input and as a gradient."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    rows, cols = shape

    def negated(*sizes):
        if sizes == (1, 1):
            view = torch.randn(sizes, generator=gen, dtype=torch.complex64, device=DEV).conj().imag
        else:
            view = torch._neg_view(torch.randn(sizes, generator=gen, device=DEV))
        assert view.is_neg() and view.is_contiguous()
        return view

    x, w, r, g = negated(rows, cols), negated(3, cols), negated(rows, 3), negated(rows, 3)
    h = negated(rows, cols)

    def results(tensors, grads):
        xs, ws, rs = (t.detach().requires_grad_() for t in tensors)
        y = linear(xs, ws, residual=rs)
        n = layer_norm(xs, ws[0])
        return [y.detach(), n.detach(), *torch.autograd.grad(y, [xs, ws], grads[0]),
                *torch.autograd.grad(n, [xs, ws], grads[1]), *checkpoint_int8(xs)]

    mine = results((x, w, r), (g, h))
    plain = results([t.resolve_neg() for t in (x, w, r)], [t.resolve_neg() for t in (g, h)])
    for a, e in zip(mine, plain):
        assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_reference_backend_launches_no_kernel_of_the_library(dtype, monkeypatch):
    """A checkpointed call too; its codes on the device are the kernels' codes."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((60, 100), generator=gen, device=DEV)
    x *= torch.exp2(torch.randint(-40, 12, (60, 1), generator=gen, device=DEV).float())
    x = x.to(dtype)
    info = torch.finfo(dtype)
    x[0], x[1], x[2], x[3] = 0.0, info.max, info.smallest_normal / 4, -63.5
    x[4, 7], x[5, 99] = math.inf, math.nan
    w = torch.randn((12, 100), generator=gen, device=DEV).to(dtype)
    codes, scales = checkpoint_int8(x)

    def refuse(*args):
        raise AssertionError("the HIP library is called")

    monkeypatch.setattr(linear_module, "require_native", refuse)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = linear(xs, ws, checkpoint="int8", backend="reference")
    dx, dw = torch.autograd.grad(out, [xs, ws], torch.ones_like(out))
    # (float16's largest number and 59 others may add up to an infinity)
    assert dw[:, :32].isnan().all() and dw[:, 96:].isnan().all() and not dw[:, 32:96].isnan().any()
    assert dx.isfinite().all()
    mine = linear_module._checkpoint_pytorch(x)
    assert torch.equal(mine[0], codes) and torch.equal(mine[1], scales)


@pytest.mark.parametrize("backend", ["auto", "reference"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_autocast_changes_nothing(checkpoint, backend):
    gen = torch.Generator(device=DEV).manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen, device=DEV) for s in ((60, 40), (24, 40), (24,)))

    def step(dtype, mode):
        leaves = [t.to(dtype, copy=True).requires_grad_() for t in (x, w, b)]
        with mode:
            out = linear(*leaves, activation="gelu", checkpoint=checkpoint, backend=backend)
            norm = layer_norm(out, leaves[2].float(), leaves[2].float(), backend=backend)
        # torch asks for backward passes outside of autocast
        return [out, norm, *torch.autograd.grad(norm.sum() + out.sum(), leaves)]

    for dtype in (torch.float32, torch.bfloat16):
        want = step(dtype, nullcontext())
        for a, e in zip(step(dtype, torch.autocast("cuda", dtype=torch.float16)), want):
            assert a.dtype == dtype and torch.equal(a, e)


@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2), (0, 1, 2)], ids=str)
def test_a_backward_allocates_for_the_wanted_gradients(which, activation):
    """A frozen weight's partial sums (33 MB here) are not allocated; every set of gradients
    equals the same ones of the whole set."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    rows, inner, outer = 40000, 512, 256
    x, w, b, g = (torch.randn(s, generator=gen, device=DEV).bfloat16()
                  for s in ((rows, inner), (outer, inner), (outer,), (rows, outer)))

    def step(which):
        leaves = [t.detach() for t in (x, w, b)]
        for i in which:
            leaves[i] = leaves[i].clone().requires_grad_()
        out = linear(*leaves, activation=activation)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(out, [leaves[i] for i in which], g)
        return grads, torch.cuda.max_memory_allocated() - before

    every, _ = step((0, 1, 2))
    grads, peak = step(which)
    for i, grad in zip(which, grads):
        assert torch.equal(grad, every[i])
    room = sum(t.numel() * 2 for t in grads) + 4 * 64 * outer * (inner * (1 in which) + 1)
    if activation == "gelu":
        room += 2 * rows * outer * 2
    assert peak <= room + (1 << 20)


def block(x, w, v, scale, checkpoint):
    hidden = linear(layer_norm(x, scale, scale), w, activation="gelu", checkpoint=checkpoint)
    return linear(hidden, v, residual=x, checkpoint=checkpoint)


@pytest.mark.parametrize("last", ["linear", "layer_norm"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_recomputed_and_offloaded_blocks(checkpoint, last):
    """A block under torch.utils.checkpoint (which ends its second forward by an exception from
    the last tensor kept) and with its kept tensors in host memory equals the plain one."""
    from torch.utils.checkpoint import checkpoint as recomputed

    gen = torch.Generator(device=DEV).manual_seed(7)
    shapes = ((500, 64), (128, 64), (64, 128), (64,))
    tensors = [torch.randn(s, generator=gen, device=DEV).bfloat16() for s in shapes]
    g = torch.randn((500, 64), generator=gen, device=DEV).bfloat16()

    def function(x, w, v, scale):
        out = block(x, w, v, scale, checkpoint)
        return out if last == "linear" else layer_norm(out, scale)

    def step(call):
        leaves = [t.clone().requires_grad_() for t in tensors]
        out = call(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = step(function)
    with torch.autograd.graph.save_on_cpu():
        offloaded = step(function)
    for got in (step(lambda *leaves: recomputed(function, *leaves, use_reentrant=False)), offloaded):
        for a, e in zip(got, want):
            assert torch.equal(a, e)
    leaves = [t.clone().requires_grad_() for t in tensors]
    recomputed(function, *leaves, use_reentrant=True).backward(g)
    for a, e in zip(leaves, want[1:]):
        assert torch.equal(a.grad, e)


def test_what_cannot_be_read_is_refused():
    """Batched tensors (vmap, gradients taken in a batch) and tensors of torch.func's
    transforms have no memory of their own: an error, not an answer."""
    x, w = torch.randn((3, 5, 8), device=DEV), torch.randn((4, 8), device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: linear(t, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layer_norm(t).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: linear(t, w), (x,), (x,))
    xs = x.clone().requires_grad_()
    out = linear(xs, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, [xs], torch.ones((2, *out.shape), device=DEV), is_grads_batched=True)


@pytest.mark.parametrize("backend", ["auto", "reference"])
@pytest.mark.parametrize(("shape", "outer"), [((0, 40), 6), ((2, 0, 5), 6), ((0, 0), 6), ((3, 0), 6),
                                              ((0,), 6), ((3, 40), 0), ((0, 40), 0), ((40,), 6)], ids=str)
def test_empty_checkpointed_calls(shape, outer, backend):
    x = torch.ones(shape, device=DEV, requires_grad=True)
    w, b = (torch.ones(s, device=DEV, requires_grad=True) for s in ((outer, shape[-1]), (outer,)))
    out = linear(x, w, b, activation="gelu", checkpoint="int8", backend=backend)
    assert out.shape == (*shape[:-1], outer)
    dx, dw, db = torch.autograd.grad(out, [x, w, b], torch.ones_like(out))
    assert dx.shape == shape and dw.shape == w.shape and db.shape == b.shape
    if 0 in shape:
        assert not dw.any() and not dx.any()
    codes, scales = checkpoint_int8(x)
    restored = checkpoint_restore(codes, scales, shape[-1], torch.float32)
    assert torch.equal(restored, x.detach().reshape(restored.shape))
