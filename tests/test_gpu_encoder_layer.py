"""A BEV encoder layer's step from the framework's operators alone, as they are used
together: projections, deformable attention, output projection with the layer's
input, norms and the feed-forward block, forward and backward, against the same
layer in PyTorch operations in float64 on the CPU."""

import pytest
import torch
import torch.nn.functional as F

from muspace_amd import layer_norm, linear, multi_scale_deformable_attn_softmax
from oracle import msda_torch

pytestmark = pytest.mark.gpu

HEADS, CHANNELS, POINTS, WIDTH, HIDDEN = 4, 16, 4, 64, 128
LEVELS = ((12, 16), (6, 8))
DEV = "cuda"


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
        "up.w": matrix(HIDDEN, WIDTH), "up.b": vector(HIDDEN),
        "down.w": matrix(WIDTH, HIDDEN), "down.b": vector(WIDTH),
        "norm2.w": vector(WIDTH, 1.0), "norm2.b": vector(WIDTH),
    }


def geometry(queries, device, dtype):
    shapes = torch.tensor(LEVELS, dtype=torch.int64, device=device)
    starts = torch.tensor([0, LEVELS[0][0] * LEVELS[0][1]], dtype=torch.int64, device=device)
    index = torch.arange(queries, device=device, dtype=dtype)
    centre = torch.stack([(index % 10 + 0.5) / 10, (index // 10 + 0.5) / (queries // 10 + 1)], -1)
    return shapes, starts, centre.view(1, queries, 1, 1, 1, 2)


def locations(offsets, centre, shapes):
    batch, queries = offsets.shape[:2]
    scale = shapes.flip(-1).to(offsets.dtype).view(1, 1, 1, len(LEVELS), 1, 2)
    return centre + offsets.view(batch, queries, HEADS, len(LEVELS), POINTS, 2) / scale


def layer(query, memory, p, checkpoint):
    # locations and logits in float32 next to a 16-bit value
    shapes, starts, centre = geometry(query.shape[1], query.device, torch.float32)
    value = linear(memory, p["value.w"], p["value.b"], checkpoint=checkpoint)
    offsets = linear(query, p["offset.w"], p["offset.b"], checkpoint=checkpoint)
    logits = linear(query, p["logit.w"], p["logit.b"], checkpoint=checkpoint)
    batch, queries = query.shape[:2]
    attended = multi_scale_deformable_attn_softmax(
        value.view(batch, -1, HEADS, CHANNELS), shapes, starts, locations(offsets.float(), centre, shapes),
        logits.float().view(batch, queries, HEADS, len(LEVELS), POINTS))
    x = linear(attended, p["out.w"], p["out.b"], residual=query, checkpoint=checkpoint)
    x = layer_norm(x, p["norm1.w"], p["norm1.b"])
    hidden = linear(x, p["up.w"], p["up.b"], activation="relu", checkpoint=checkpoint)
    x = linear(hidden, p["down.w"], p["down.b"], residual=x, checkpoint=checkpoint)
    return layer_norm(x, p["norm2.w"], p["norm2.b"])


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
    x = F.linear(attended, p["out.w"], p["out.b"]) + query
    x = F.layer_norm(x, (WIDTH,), p["norm1.w"], p["norm1.b"])
    x = F.linear(F.relu(F.linear(x, p["up.w"], p["up.b"])), p["down.w"], p["down.b"]) + x
    return F.layer_norm(x, (WIDTH,), p["norm2.w"], p["norm2.b"])


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_step(dtype, checkpoint):
    gen = torch.Generator().manual_seed(11)
    batch, queries = 2, 190
    spatial = sum(h * w for h, w in LEVELS)
    tensors = {"query": torch.randn((batch, queries, WIDTH), generator=gen),
               "memory": torch.randn((batch, spatial, WIDTH), generator=gen), **parameters(gen)}
    tensors = {k: v.to(dtype) for k, v in tensors.items()}
    grad = torch.randn((batch, queries, WIDTH), generator=gen).to(dtype)

    mine = {k: v.to(DEV).requires_grad_() for k, v in tensors.items()}
    out = layer(mine["query"], mine["memory"], mine, checkpoint)
    out.backward(grad.to(DEV))
    exact = {k: v.double().requires_grad_() for k, v in tensors.items()}
    expected = plain_layer(exact["query"], exact["memory"], exact)
    expected.backward(grad.double())

    # relative to each tensor's root mean square. A rounding to the type is half a step
    # (2^-24, 2^-9) at most and passes about ten operators here; a location or a
    # pre-activation that falls on the other side of a cell's border or of zero moves
    # single elements, so the measure is the mean. A checkpoint's step is under
    # top / 63.5, top the block's largest magnitude, since 127 half steps do not reach it;
    # errors of a step's even spread have a root mean square of step / sqrt(12), under
    # top / 219. In 32 normal values top is 2.4 standard deviations on average, 3 at times,
    # and of rectified ones (the hidden layer) 1.41 times that against their own root mean
    # square: 3.4 / 219 < 2^-6. Errors of different rows are independent, as the terms
    # of the weight's gradient are, so that its relative error is theirs.
    def distance(a, e):
        return float((a.detach().cpu().double() - e.detach()).square().mean().sqrt()
                     / e.detach().square().mean().sqrt())

    base = 40 * 2.0**-9 if dtype == torch.bfloat16 else 2.0**-12
    assert distance(out, expected) <= base / 2
    for name, leaf in mine.items():
        limit = base
        if checkpoint and name.endswith(".w") and not name.startswith("norm"):
            limit += 2.0**-6
        assert leaf.grad is not None and leaf.grad.dtype == dtype, name
        # offsets' gradients are differences of neighbouring cells' values
        factor = 2 if name.startswith(("offset", "logit", "query", "memory", "value")) else 1
        assert distance(leaf.grad, exact[name].grad) <= factor * limit, name
