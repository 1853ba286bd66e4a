"""Measured cases of the encoder layer's dense operators.

A deformable-attention encoder or decoder layer is the attention operator,
projections around it, a feed-forward block and layer norms. The cases run the
dense part through the public operators of ``muspace_amd`` (inference: the
call; training: the call and its gradients):

  linear      ``linear``: act(x W^T + b) + residual, gradients of x, W, b and
              the residual
  checkpoint  ``linear`` with ``checkpoint="int8"``: the backward reads the
              input from 8-bit codes, blocks of 32 values that share a power of
              two
  layer_norm  ``layer_norm`` over the last dimension, gradients of x, weight
              and bias

With ``own`` false, ``run`` computes the same from elementary torch operations
in float32.

Inputs and weights lie on grids coarse enough for every partial sum of x W^T + b
to be a float32 number, so each side sees the same pre-activations: the
derivative of relu jumps at zero, and a pre-activation next to it would
otherwise fall on either side by the order of a sum.
"""

from __future__ import annotations

import math

import torch

own = False  # set from outside: the framework's operators instead of the plain form

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5
BLOCK = 32  # values of a row that share a scale in an 8-bit checkpoint


def _linear(name, mode, dtype, rows, inner, outer, activation="none", residual=False,
            checkpoint=False):
    return {"name": name, "op": "checkpoint" if checkpoint else "linear", "mode": mode,
            "dtype": dtype, "rows": rows, "in": inner, "out": outer, "activation": activation,
            "residual": residual}


def _norm(name, mode, dtype, rows, inner):
    return {"name": name, "op": "layer_norm", "mode": mode, "dtype": dtype, "rows": rows,
            "in": inner}


def listed():
    return [
        # output projection of an object decoder's attention while serving one
        # image: 300 queries, the layer's input added; the latency of a call
        _linear("decoder_out_infer_f16", "infer", "float16", 300, 256, 256, residual=True),
        # first product of a BEV encoder's feed-forward block, inference
        _linear("bev_ffn_in_infer_bf16", "infer", "bfloat16", 40000, 256, 512, "relu"),
        # the same of an image encoder over four levels, two images, training
        _linear("encoder_ffn_in_train_f32", "train", "float32", 44446, 256, 1024, "relu"),
        # second product of the BEV block with its residual, two samples, training
        _linear("bev_ffn_out_train_bf16", "train", "bfloat16", 80000, 512, 256, residual=True),
        # a block of odd widths, rows off every alignment, training
        _linear("odd_ffn_train_f16", "train", "float16", 30021, 203, 611, "gelu"),
        # value projection of spatial cross-attention, two samples of six
        # cameras with four levels: the most rows a layer has
        _linear("value_proj_train_bf16", "train", "bfloat16", 369900, 256, 256),
        # the BEV block's first product, its input kept in 8 bits
        _linear("bev_ffn_in_checkpoint_train_bf16", "train", "bfloat16", 40000, 256, 512, "relu",
                checkpoint=True),
        # a decoder block's second product in float32, its input in 8 bits
        _linear("decoder_ffn_out_checkpoint_train_f32", "train", "float32", 1800, 1024, 256,
                residual=True, checkpoint=True),
        # norms: a decoder layer while serving, ...
        _norm("decoder_norm_infer_f16", "infer", "float16", 300, 256),
        # ... an image encoder's in training, ...
        _norm("encoder_norm_train_f32", "train", "float32", 44446, 256),
        # ... odd width, rows off every alignment, ...
        _norm("odd_norm_train_f16", "train", "float16", 30021, 611),
        # ... and the queries of twelve cameras
        _norm("camera_norm_train_bf16", "train", "bfloat16", 180000, 256),
    ]


MAX_FLOPS = 6 * 369900 * 256 * 256  # the largest listed products, all three of a training step
MAX_FLOPS_F32 = 6 * 44446 * 256 * 1024
MAX_ELEMENTS = 369900 * 256  # rows of an input or output
MAX_NORM_ELEMENTS = 180000 * 256


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_width(rng, low, high):
    width = _log_uniform(rng, low, high)
    kind = rng.random()
    if kind < 0.5:  # the widths of most models
        return max(32, (width + 16) // 32 * 32)
    if kind < 0.75:
        return max(8, width // 8 * 8)
    return width


def draw(rng):
    op = rng.choice(["linear", "linear", "checkpoint", "layer_norm"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    mode = "train" if op == "checkpoint" else rng.choice(["infer", "train"])
    while True:
        rows = _log_uniform(rng, 1, 369900)
        inner = _draw_width(rng, 32, 2048)
        if op == "layer_norm":
            if rows * inner <= MAX_NORM_ELEMENTS // (2 if dtype == "float32" else 1):
                return {"op": op, "mode": mode, "dtype": dtype, "rows": rows, "in": inner}
            continue
        outer = _draw_width(rng, 32, 2048)
        flops = (6 if mode == "train" else 2) * rows * inner * outer
        if (flops <= (MAX_FLOPS_F32 if dtype == "float32" else MAX_FLOPS)
                and rows * max(inner, outer) <= MAX_ELEMENTS // (2 if dtype == "float32" else 1)):
            return {"op": op, "mode": mode, "dtype": dtype, "rows": rows, "in": inner,
                    "out": outer, "activation": rng.choice(["none", "relu", "relu", "gelu"]),
                    "residual": rng.random() < 0.4}


def work(case):
    """Each input read once, each output written once; the residual's gradient
    is the output's own and is not written."""
    width = 4 if case["dtype"] == "float32" else 2
    rows, inner, train = case["rows"], case["in"], case["mode"] == "train"
    if case["op"] == "layer_norm":
        values = rows * inner * (4 if train else 2) + inner * (4 if train else 2)
        return {"bytes": width * values, "flops": rows * inner * (20 if train else 8)}
    outer = case["out"]
    values = rows * (inner + outer * (2 if case["residual"] else 1)) + outer * inner + outer
    if train:
        values += rows * (inner + outer) + outer * inner + outer
    return {"bytes": width * values, "flops": (6 if train else 2) * rows * inner * outer}


# ------------------------------------------------------------- inputs ---


def _grid(values, step, limit):
    return torch.round(values / step).mul_(step).clamp_(-limit, limit)


def _inputs(case, seed):
    """A case's tensors, before any requires a gradient."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows, inner = case["rows"], case["in"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    if case["op"] == "layer_norm":
        # a residual stream: every channel with a spread and an offset of its own
        spread = torch.exp(0.5 * normal(inner))
        tensors = {"x": (normal(rows, inner) * spread + 0.5 * normal(inner)).to(dtype),
                   "weight": (1.0 + 0.2 * normal(inner)).to(dtype),
                   "bias": (0.2 * normal(inner)).to(dtype)}
        if case["mode"] == "train":
            tensors["grad"] = normal(rows, inner).to(dtype)
        return tensors
    outer = case["out"]
    # steps that each type holds exactly: x of 7 (bfloat16) or 10 bits, weights of
    # 7 or 8; with |weight| <= 2^-e a sum stays under 2^24 steps up to |sum| = 8
    fine = 0 if dtype is torch.bfloat16 else 1
    e = math.ceil(math.log2(math.sqrt(inner)))
    x_step, w_step = 2.0 ** -(4 + 3 * fine), 2.0 ** -(7 + fine + e)
    x = _grid(normal(rows, inner), x_step, 7.5)
    bound = 1.0 / math.sqrt(inner)

    def uniform(*shape):
        values = torch.rand(shape, generator=gen, device=DEVICE) * (2 * bound) - bound
        return _grid(values, w_step, 2.0 ** -e)

    tensors = {"x": x.to(dtype), "weight": uniform(outer, inner).to(dtype),
               "bias": uniform(outer).to(dtype)}
    if case["residual"]:
        tensors["residual"] = normal(rows, outer).to(dtype)
    if case["mode"] == "train":
        tensors["grad"] = normal(rows, outer).to(dtype)
    return tensors


def _leaves(case):
    names = ["x", "weight", "bias"]
    if case.get("residual"):
        names.append("residual")
    return names


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["mode"] == "train":
        for name in _leaves(case):
            state[name].requires_grad_()
    state["case"] = case
    return state


# ---------------------------------------------------------- operators ---


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            return _plain_layer_norm(case, state)
        return _plain_linear(case, state)


def _run_own(case, state):
    from muspace_amd import layer_norm, linear

    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "layer_norm":
            out = layer_norm(state["x"], state["weight"], state["bias"], eps=EPS)
        else:
            activation = None if case["activation"] == "none" else case["activation"]
            checkpoint = "int8" if case["op"] == "checkpoint" else None
            out = linear(state["x"], state["weight"], state["bias"], activation=activation,
                         residual=state.get("residual"), checkpoint=checkpoint)
    if not train:
        return [out]
    leaves = [state[name] for name in _leaves(case)]
    return [out.detach(), *torch.autograd.grad(out, leaves, state["grad"])]


def _plain_layer_norm(case, state):
    dtype = state["x"].dtype
    x, weight, bias = state["x"].float(), state["weight"].float(), state["bias"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    out = (xhat * weight + bias).to(dtype)
    if case["mode"] != "train":
        return [out]
    grad = state["grad"].float()
    gw = grad * weight
    grad_x = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    return [out, grad_x.to(dtype), (grad * xhat).sum(0).to(dtype), grad.sum(0).to(dtype)]


def _read_back(x):
    """x as its 8-bit checkpoint holds it: blocks of 32 along a row, codes of
    -127..127 times the smallest power of two that reaches the block's largest."""
    rows, inner = x.shape
    pad = -inner % BLOCK
    blocks = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    exponent = exponent - 7 + (mantissa > 127.0 / 128.0).to(exponent.dtype)
    scale = torch.ldexp(torch.ones_like(mantissa), exponent.clamp_min(-24))
    return (torch.round(blocks / scale) * scale).view(rows, -1)[:, :inner]


def _plain_linear(case, state):
    dtype = state["x"].dtype
    x, weight, bias = state["x"].float(), state["weight"].float(), state["bias"].float()
    z = x @ weight.t() + bias
    slope = None
    if case["activation"] == "relu":
        out, slope = torch.clamp_min(z, 0.0), (z > 0).float()
    elif case["activation"] == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        out = z * cdf
        slope = cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    else:
        out = z
    if case["residual"]:
        out = out + state["residual"].float()
    out = out.to(dtype)
    if case["mode"] != "train":
        return [out]
    dz = state["grad"].float()
    if slope is not None:
        dz = dz * slope
    kept = _read_back(x) if case["op"] == "checkpoint" else x
    grads = [(dz @ weight).to(dtype), (dz.t() @ kept).to(dtype), dz.sum(0).to(dtype)]
    if case["residual"]:
        grads.append(state["grad"])
    return [out, *grads]


# ------------------------------------------------------------- 64 bits ---


def exact(case, seed):
    tensors = {name: value.double() for name, value in _inputs(case, seed).items()}
    x, weight, bias = tensors["x"], tensors["weight"], tensors["bias"]
    grad = tensors.get("grad")
    if case["op"] == "layer_norm":
        mean = x.sum(-1, keepdim=True) / x.shape[-1]
        sigma = ((x - mean).square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        unit = (x - mean) / sigma
        out = [unit * weight + bias]
        if grad is not None:
            scaled = grad * weight
            along = (scaled * unit).sum(-1, keepdim=True) / x.shape[-1]
            level = scaled.sum(-1, keepdim=True) / x.shape[-1]
            out += [(scaled - level - unit * along) / sigma, (grad * unit).sum(0), grad.sum(0)]
        return out
    z = torch.addmm(bias, x, weight.t())
    if case["activation"] == "relu":
        y, dz = z.clamp_min(0.0), None if grad is None else grad.masked_fill(z <= 0, 0.0)
    elif case["activation"] == "gelu":
        half = torch.erfc(z * -math.sqrt(0.5)) / 2
        density = torch.exp(z.square() / -2) / math.sqrt(2 * math.pi)
        y, dz = z * half, None if grad is None else grad * (half + z * density)
    else:
        y, dz = z, grad
    if case["residual"]:
        y = y + tensors["residual"]
    if grad is None:
        return [y]
    if case["op"] == "checkpoint":
        rows, inner = x.shape
        kept = torch.zeros_like(x)
        for first in range(0, inner, BLOCK):
            part = x[:, first:first + BLOCK]
            top = part.abs().amax(1, keepdim=True).clamp_min(2.0 ** -40)
            power = torch.ceil(torch.log2(top / 127.0))
            # log2 rounds: step to the smallest power that reaches the top
            power += (torch.exp2(power) * 127.0 < top).double()
            power -= (torch.exp2(power - 1) * 127.0 >= top).double()
            scale = torch.exp2(power.clamp_min(-24.0))
            kept[:, first:first + BLOCK] = torch.round(part / scale) * scale
        x = kept
    out = [y, dz @ weight, dz.t() @ x, dz.sum(0)]
    if case["residual"]:
        out.append(grad)
    return out
