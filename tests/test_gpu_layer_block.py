"""A layer that norms before its blocks, from the framework's operators as they are used
together: deformable attention, its output dropped out, summed and normed in one, a gated
feed-forward block with dropout inside, its norm, gate and sum; forward and backward against the
same in float64 on the CPU. And the same layer deployed, its products in 8-bit integers."""

import pytest
import torch
import torch.nn.functional as F

from muspace_amd import (
    dropout,
    gated_linear,
    linear,
    linear_int8,
    multi_scale_deformable_attn_softmax,
    quantize_int8,
    residual_norm,
)
from oracle import block_torch, msda_torch
from test_gpu_encoder_layer import CHANNELS, HEADS, LEVELS, POINTS, WIDTH, geometry, locations

pytestmark = pytest.mark.gpu

DEV = "cuda"
HIDDEN, P, SEED = 96, 0.1, 123
BATCH, QUERIES = 2, 190


def parameters(gen):
    def matrix(outer, inner):
        return torch.randn((outer, inner), generator=gen) / inner**0.5

    def vector(n, centre=0.0):
        return centre + 0.1 * torch.randn(n, generator=gen)

    samples = HEADS * len(LEVELS) * POINTS
    return {
        "value.w": matrix(WIDTH, WIDTH), "value.b": vector(WIDTH),
        "offset.w": matrix(2 * samples, WIDTH) * 0.5, "offset.b": vector(2 * samples),
        "logit.w": matrix(samples, WIDTH), "logit.b": vector(samples),
        "out.w": matrix(WIDTH, WIDTH), "out.b": vector(WIDTH),
        "norm1.w": vector(WIDTH, 1.0), "norm1.b": vector(WIDTH),
        "up.w": matrix(2 * HIDDEN, WIDTH), "up.b": vector(2 * HIDDEN),
        "down.w": matrix(WIDTH, HIDDEN), "down.b": vector(WIDTH),
        "post.w": vector(WIDTH, 1.0), "gate": vector(WIDTH, 0.5),
        "norm2.w": vector(WIDTH, 1.0), "norm2.b": vector(WIDTH),
    }


def layer(query, memory, p, seed, product=linear, dropout_p=P, fixed=None):
    """(normed, stream); ``product``: of the dense layers after the attention; ``fixed``: the
    geometry, which a capture may not copy from the host."""
    shapes, starts, centre = fixed or geometry(query.shape[1], query.device, torch.float32)
    value = linear(memory, p["value.w"], p["value.b"])
    offsets = linear(query, p["offset.w"], p["offset.b"])
    logits = linear(query, p["logit.w"], p["logit.b"])
    batch, queries = query.shape[:2]
    attended = multi_scale_deformable_attn_softmax(
        value.view(batch, -1, HEADS, CHANNELS), shapes, starts, locations(offsets.float(), centre, shapes),
        logits.float().view(batch, queries, HEADS, len(LEVELS), POINTS))
    out = product(attended, p["out.w"], p["out.b"])
    normed, stream = residual_norm(out, query, p["norm1.w"], p["norm1.b"], dropout_p=dropout_p,
                                   seed=seed, offset=0)
    hidden = gated_linear(normed, p["up.w"], p["up.b"], activation="silu")
    hidden = dropout(hidden, dropout_p, seed=seed, offset=1)
    out = product(hidden, p["down.w"], p["down.b"])
    return residual_norm(out, stream, p["norm2.w"], p["norm2.b"], post_norm="rms",
                         post_weight=p["post.w"], gate=p["gate"], dropout_p=dropout_p, seed=seed,
                         offset=2)


def plain_layer(query, memory, p):
    shapes, _, centre = geometry(query.shape[1], query.device, query.dtype)
    value = F.linear(memory, p["value.w"], p["value.b"])
    offsets = F.linear(query, p["offset.w"], p["offset.b"])
    logits = F.linear(query, p["logit.w"], p["logit.b"])
    batch, queries = query.shape[:2]
    weights = logits.view(batch, queries, HEADS, -1).softmax(-1)
    attended = msda_torch.msda_forward(
        value.view(batch, -1, HEADS, CHANNELS), shapes, locations(offsets, centre, shapes),
        weights.view(batch, queries, HEADS, len(LEVELS), POINTS))

    def drop(x, offset):
        kept = block_torch.kept(0, x.numel(), P, SEED, offset).view(x.shape)
        return x * kept / (1 - P)

    stream = query + drop(F.linear(attended, p["out.w"], p["out.b"]), 0)
    normed = F.layer_norm(stream, (WIDTH,), p["norm1.w"], p["norm1.b"])
    a, u = F.linear(normed, p["up.w"], p["up.b"]).chunk(2, -1)
    out = F.linear(drop(F.silu(a) * u, 1), p["down.w"], p["down.b"])
    out = out / (out.square().mean(-1, keepdim=True) + 1e-5).sqrt() * p["post.w"]
    stream = stream + p["gate"] * drop(out, 2)
    return F.layer_norm(stream, (WIDTH,), p["norm2.w"], p["norm2.b"]), stream


def draw(dtype):
    gen = torch.Generator().manual_seed(11)
    spatial = sum(h * w for h, w in LEVELS)
    tensors = {"query": torch.randn((BATCH, QUERIES, WIDTH), generator=gen),
               "memory": torch.randn((BATCH, spatial, WIDTH), generator=gen), **parameters(gen)}
    grads = [torch.randn((BATCH, QUERIES, WIDTH), generator=gen).to(dtype) for _ in range(2)]
    return {k: v.to(dtype) for k, v in tensors.items()}, grads


def distance(a, e):
    return float((a.detach().cpu().double() - e.detach()).square().mean().sqrt()
                 / e.detach().square().mean().sqrt())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_step(dtype):
    tensors, grads = draw(dtype)
    mine = {k: v.to(DEV).requires_grad_() for k, v in tensors.items()}
    seed = torch.tensor([SEED], device=DEV)  # as a captured step would hold it
    outs = layer(mine["query"], mine["memory"], mine, seed)
    torch.autograd.backward(outs, [g.to(DEV) for g in grads])
    exact = {k: v.double().requires_grad_() for k, v in tensors.items()}
    expected = plain_layer(exact["query"], exact["memory"], exact)
    torch.autograd.backward(expected, [g.double() for g in grads])
    # relative to each tensor's root mean square: about ten operators round to half a step
    # (2^-24, 2^-9) at most each, in either direction; a location that falls on the other side of
    # a cell's border moves single elements, so the measure is the mean
    base = 40 * 2.0**-9 if dtype == torch.bfloat16 else 2.0**-12
    for a, e in zip(outs, expected):
        assert distance(a, e) <= base / 2
    for name, leaf in mine.items():
        assert leaf.grad is not None and leaf.grad.dtype == dtype, name
        # offsets' gradients are differences of neighbouring cells' values
        factor = 2 if name.startswith(("offset", "logit", "query", "memory", "value")) else 1
        assert distance(leaf.grad, exact[name].grad) <= factor * base, name


def test_captured_steps_draw_new_masks():
    """Forward and backward in one graph; the seed's tensor counts on between replays."""
    tensors, grads = draw(torch.bfloat16)
    mine = {k: v.to(DEV).requires_grad_() for k, v in tensors.items()}
    grads = [g.to(DEV) for g in grads]
    seed = torch.tensor([SEED], device=DEV)
    fixed = geometry(QUERIES, torch.device(DEV), torch.float32)

    def step(seed):
        outs = layer(mine["query"], mine["memory"], mine, seed, fixed=fixed)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, list(mine.values()), grads)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(seed)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(seed)
    # grad_value's sums at tile borders are added in no fixed order, so what is made of it alone is
    # the same up to rounding: each run is within 2 * 40 * 2^-9 of float64 (test_layer_step), two
    # runs within 4 * 40 * 2^-9 of each other
    unordered = ("memory", "value.w", "value.b")
    seen = []
    for replay in range(1, 4):
        seed.add_(1)
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        for name, a, e in zip(("normed", "stream", *mine), got, step(SEED + replay)):
            if name in unordered:
                assert distance(a, e.cpu().double()) <= 4 * 40 * 2.0**-9, name
            else:
                assert torch.equal(a, e), name
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.parametrize("queries", [1, QUERIES])
def test_deployed_layer(queries):
    """No dropout, no gradients, the products after the attention in 8-bit integers: codes of rows
    of n values err by a step of top / 127 evenly spread, under 3.5 / 127 / sqrt(12) = 2^-7 of the
    values' root mean square for rows and weights each, and the norms and the sum pass it on."""
    tensors, _ = draw(torch.bfloat16)
    p = {k: v.to(DEV) for k, v in tensors.items()}
    codes = {k: quantize_int8(p[k]) for k in ("out.w", "down.w")}
    by_weight = {id(p[k]): codes[k] for k in codes}

    def product(x, weight, bias):
        return linear_int8(x, *by_weight[id(weight)], bias)

    query = p["query"][:, :queries]
    with torch.no_grad():
        want = layer(query, p["memory"], p, None, dropout_p=0.0)
        got = layer(query, p["memory"], p, None, product=product, dropout_p=0.0)
    for a, e in zip(got, want):
        assert a.shape == query.shape
        assert distance(a, e.cpu().double()) <= 4 * 2.0**-7
        assert not torch.equal(a, e)
