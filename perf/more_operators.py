"""Measured cases of a transformer layer's other dense steps.

Next to the products and norms that ``perf/operators.py`` measures, a layer of an
image encoder, a BEV encoder or an object decoder has a feed-forward block that may
be gated, dropout while it is trained, the sum of each block with the residual
stream and the norm that follows, and, once deployed, products in 8-bit integers.
The cases run them through the public operators of ``muspace_amd`` (inference: the
call; training: the call and its gradients):

  gated      ``gated_linear``: act(x Wg^T + bg) * (x Wu^T + bu), the weights packed
             [Wg; Wu], gradients of x, weight and bias
  dropout    ``dropout``: a mask from a counter-based generator that no tensor
             holds, optionally added to the residual stream, and its gradients
  block      ``residual_norm``: stream = scale * residual + gate * dropout(
             post_norm(block)), then the next norm; gradients of all of it
  int8       ``linear_int8``: rows of x quantised to 8 bits with a scale each,
             multiplied with a weight of 8-bit rows (``quantize_int8``)

With ``own`` false, ``run`` computes the same from elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False  # set from outside: the framework's operators instead of the plain form

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5


def _gated(name, mode, dtype, rows, inner, hidden, activation="silu"):
    return {"name": name, "op": "gated", "mode": mode, "dtype": dtype, "rows": rows, "in": inner,
            "hidden": hidden, "activation": activation}


def _dropout(name, dtype, rows, inner, p=0.1, residual=True):
    return {"name": name, "op": "dropout", "mode": "train", "dtype": dtype, "rows": rows,
            "in": inner, "p": p, "residual": residual}


def _block(name, mode, dtype, rows, inner, norm="layer", post="none", gate=False, scale=1.0,
           p=0.0):
    return {"name": name, "op": "block", "mode": mode, "dtype": dtype, "rows": rows, "in": inner,
            "norm": norm, "post": post, "gate": gate, "scale": scale, "p": p}


def _int8(name, dtype, rows, inner, outer, activation="none", residual=False):
    return {"name": name, "op": "int8", "mode": "infer", "dtype": dtype, "rows": rows,
            "in": inner, "out": outer, "activation": activation, "residual": residual}


def listed():
    return [
        # a single token while serving: reading the weights is all of it
        _gated("token_gated_infer_bf16", "infer", "bfloat16", 1, 1024, 4096),
        # a BEV encoder's feed-forward block, gated, in training
        _gated("bev_gated_train_bf16", "train", "bfloat16", 40000, 256, 512),
        # odd widths, rows off every alignment, float32
        _gated("odd_gated_train_f32", "train", "float32", 30021, 203, 611, "gelu"),
        # a wide block, bound by its products
        _gated("wide_gated_train_bf16", "train", "bfloat16", 16384, 1024, 4096),
        # dropout of a feed-forward block's hidden values, odd width
        _dropout("odd_dropout_train_f16", "float16", 30021, 611, residual=False),
        # dropout of the attention's output over twelve cameras' queries, added to
        # the queries
        _dropout("camera_dropout_add_train_bf16", "bfloat16", 180000, 256),
        # end of a decoder layer's block while serving one image: 300 queries
        _block("decoder_add_norm_infer_f16", "infer", "float16", 300, 256),
        # an image encoder's over four levels, two images, with dropout
        _block("encoder_add_norm_train_f32", "train", "float32", 44446, 256, p=0.1),
        # norms before and after a wide block, learned gate
        _block("wide_sandwich_train_bf16", "train", "bfloat16", 20000, 1024, "rms", "rms", True,
               p=0.1),
        # a decoder's output projection in 8 bits, 300 queries
        _int8("decoder_out_int8_f16", "float16", 300, 256, 256, residual=True),
        # first product of a BEV encoder's feed-forward block in 8 bits
        _int8("bev_ffn_in_int8_bf16", "bfloat16", 40000, 256, 512, "relu"),
        # a wide product in 8 bits, bound by the matrix cores
        _int8("wide_int8_bf16", "bfloat16", 16384, 2048, 8192, "gelu"),
    ]


MAX_FLOPS = 6 * 16384 * 1024 * 2 * 4096  # the largest listed products of a training step
MAX_ELEMENTS = 180000 * 256  # of the largest tensor of rows
MAX_HIDDEN = 16384 * 8192


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
    op = rng.choice(["gated", "gated", "dropout", "block", "block", "int8"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    slow = 8 if dtype == "float32" else 1
    mode = {"dropout": "train", "int8": "infer"}.get(op) or rng.choice(["infer", "train"])
    while True:
        rows = _log_uniform(rng, 1, 180000)
        inner = _draw_width(rng, 32, 2048)
        case = {"op": op, "mode": mode, "dtype": dtype, "rows": rows, "in": inner}
        if rows * inner > MAX_ELEMENTS // (2 if dtype == "float32" else 1):
            continue
        if op == "dropout":
            return {**case, "p": round(rng.uniform(0.01, 0.6), 3), "residual": rng.random() < 0.5}
        if op == "block":
            norm = rng.choice(["layer", "rms"])
            return {**case, "norm": norm, "post": rng.choice(["none", "none", "layer", "rms"]),
                    "gate": rng.random() < 0.4, "scale": rng.choice([1.0, 1.0, 0.5, 1.7]),
                    "p": rng.choice([0.0, 0.1, round(rng.uniform(0.01, 0.6), 3)])}
        outer = _draw_width(rng, 32, 4096)
        if op == "gated":
            flops = (6 if mode == "train" else 2) * rows * inner * 2 * outer
            if flops <= MAX_FLOPS // slow and rows * 2 * outer <= MAX_HIDDEN // 2:
                return {**case, "hidden": outer,
                        "activation": rng.choice(["silu", "silu", "gelu", "sigmoid"])}
        elif rows * inner * outer <= 16384 * 2048 * 8192 // 4 and rows * outer <= MAX_HIDDEN // 2:
            return {**case, "out": outer, "activation": rng.choice(["none", "relu", "gelu"]),
                    "residual": rng.random() < 0.4}


def work(case):
    """Each input read once, each output written once."""
    width = 4 if case["dtype"] == "float32" else 2
    rows, inner, train = case["rows"], case["in"], case["mode"] == "train"
    values = rows * inner
    if case["op"] == "gated":
        hidden = case["hidden"]
        weights = 2 * hidden * (inner + 1)
        moved = rows * (inner + hidden) + weights
        return {"bytes": width * moved * (2 if train else 1),
                "flops": (6 if train else 2) * rows * inner * 2 * hidden}
    if case["op"] == "dropout":
        # x (and the residual), the output; their gradients: the residual's is the
        # output's own and is not written
        return {"bytes": width * values * (5 if case["residual"] else 4), "flops": 2 * values}
    if case["op"] == "block":
        vectors = 2 if case["norm"] == "layer" else 1
        vectors += {"none": 0, "layer": 2, "rms": 1}[case["post"]] + (1 if case["gate"] else 0)
        if not train:
            return {"bytes": width * (4 * values + vectors * inner), "flops": 12 * values}
        # forward: block, residual, stream, output; backward: the output's and the
        # stream's gradients in, the block's and the residual's out (both at once
        # where they are the same)
        same = (case["post"] == "none" and not case["gate"] and case["scale"] == 1.0
                and case["p"] == 0.0)
        return {"bytes": width * ((7 if same else 8) * values + 2 * vectors * inner),
                "flops": 30 * values}
    outer = case["out"]
    moved = width * (values + rows * outer * (2 if case["residual"] else 1) + outer)
    return {"bytes": moved + outer * inner + 4 * outer, "flops": 2 * values * outer}


# ------------------------------------------------------------- inputs ---


def _inputs(case, seed):
    """A case's tensors, before any requires a gradient."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows, inner, train = case["rows"], case["in"], case["mode"] == "train"

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    def uniform(bound, *shape):
        return torch.rand(shape, generator=gen, device=DEVICE) * (2 * bound) - bound

    def stream():
        # a residual stream: every channel with a spread and an offset of its own
        spread = torch.exp(0.5 * normal(inner))
        return (normal(rows, inner) * spread + 0.5 * normal(inner)).to(dtype)

    bound = 1.0 / math.sqrt(inner)
    if case["op"] == "gated":
        hidden = case["hidden"]
        tensors = {"x": normal(rows, inner).to(dtype),
                   "weight": (2.0 * uniform(bound, 2 * hidden, inner)).to(dtype),
                   "bias": uniform(bound, 2 * hidden).to(dtype)}
        if train:
            tensors["grad"] = normal(rows, hidden).to(dtype)
        return tensors
    if case["op"] == "dropout":
        tensors = {"x": normal(rows, inner).to(dtype)}
        if case["residual"]:
            tensors["residual"] = stream()
        tensors["grad"] = normal(rows, inner).to(dtype)
        return tensors
    if case["op"] == "block":
        tensors = {"x": normal(rows, inner).to(dtype), "residual": stream(),
                   "weight": (1.0 + 0.2 * normal(inner)).to(dtype)}
        if case["norm"] == "layer":
            tensors["bias"] = (0.2 * normal(inner)).to(dtype)
        if case["post"] != "none":
            tensors["post_weight"] = (1.0 + 0.2 * normal(inner)).to(dtype)
        if case["post"] == "layer":
            tensors["post_bias"] = (0.2 * normal(inner)).to(dtype)
        if case["gate"]:
            tensors["gate"] = (0.5 + 0.2 * normal(inner)).to(dtype)
        if train:
            tensors["grad"] = normal(rows, inner).to(dtype)
            tensors["grad_stream"] = normal(rows, inner).to(dtype)
        return tensors
    outer = case["out"]
    # activations with a few wide channels, as they are met before a product
    spread = torch.exp(0.5 * normal(inner))
    weight = uniform(bound, outer, inner)
    scale = (weight.abs().amax(-1) / 127.0).clamp_min(2.0 ** -126)
    tensors = {"x": (normal(rows, inner) * spread).to(dtype),
               "weight": torch.round(weight / scale[:, None]).to(torch.int8), "scale": scale,
               "bias": uniform(bound, outer).to(dtype)}
    if case["residual"]:
        tensors["residual"] = normal(rows, outer).to(dtype)
    return tensors


LEAVES = ("x", "residual", "weight", "bias", "post_weight", "post_bias", "gate")


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["mode"] == "train":
        state["leaves"] = [state[name].requires_grad_() for name in LEAVES if name in state]
    state["case"] = case
    state["seed"] = 77003 * seed + 12345  # of the dropout's generator
    return state


# ---------------------------------------------------------- operators ---


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "gated":
            return _plain_gated(case, state)
        if case["op"] == "dropout":
            return _plain_dropout(case, state)
        if case["op"] == "block":
            return _plain_block(case, state)
        return _plain_int8(case, state)


def _run_own(case, state):
    from muspace_amd import dropout, gated_linear, linear_int8, residual_norm

    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "gated":
            outs = [gated_linear(state["x"], state["weight"], state["bias"],
                                 activation=case["activation"])]
        elif case["op"] == "dropout":
            outs = [dropout(state["x"], case["p"], seed=state["seed"], offset=3,
                            residual=state.get("residual"))]
        elif case["op"] == "block":
            outs = residual_norm(
                state["x"], state["residual"], state["weight"], state.get("bias"),
                norm=case["norm"], eps=EPS,
                post_norm=None if case["post"] == "none" else case["post"],
                post_weight=state.get("post_weight"), post_bias=state.get("post_bias"),
                gate=state.get("gate"), residual_scale=case["scale"], dropout_p=case["p"],
                seed=state["seed"], offset=3)
        else:
            activation = None if case["activation"] == "none" else case["activation"]
            outs = [linear_int8(state["x"], state["weight"], state["scale"], state["bias"],
                                activation=activation, residual=state.get("residual"))]
    outs = list(outs)
    if not train:
        return outs
    grads = [state["grad"]]
    if case["op"] == "block":
        grads.append(state["grad_stream"])
    return [*(out.detach() for out in outs), *torch.autograd.grad(outs, state["leaves"], grads)]


def _act(a, activation):
    """The activation and its derivative."""
    if activation == "gelu":
        cdf = 0.5 * torch.erfc(a * -math.sqrt(0.5))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-a))
    if activation == "sigmoid":
        return sig, sig * (1.0 - sig)
    return a * sig, sig * (1.0 + a * (1.0 - sig))


def _plain_gated(case, state):
    dtype = state["x"].dtype
    x, weight, bias = state["x"].float(), state["weight"].float(), state["bias"].float()
    hidden = case["hidden"]
    z = x @ weight.t() + bias
    a, u = z[:, :hidden], z[:, hidden:]
    h, slope = _act(a, case["activation"])
    out = (h * u).to(dtype)
    if case["mode"] != "train":
        return [out]
    grad = state["grad"].float()
    dz = torch.cat((grad * u * slope, grad * h), -1)
    return [out, (dz @ weight).to(dtype), (dz.t() @ x).to(dtype), dz.sum(0).to(dtype)]


MASK32 = 0xFFFFFFFF


def _words(count, seed, offset):
    """Philox4x32-10: word i % 4 of counter (i // 4, offset) under the key `seed`,
    for i up to `count`; numbers of 32 bits held in 64."""
    index = torch.arange((count + 3) // 4, device=DEVICE)
    c0, c1 = index & MASK32, index >> 32
    c2, c3 = torch.full_like(index, offset & MASK32), torch.full_like(index, offset >> 32)
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(10):
        # 64-bit products wrap around; their upper halves are right all the same
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & MASK32 ^ c1 ^ k0, p1 & MASK32,
                          (p0 >> 32) & MASK32 ^ c3 ^ k1, p0 & MASK32)
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack((c0, c1, c2, c3), -1).view(-1)[:count]


def _factor(case, state):
    """What dropout multiplies each value with: 0 or 1 / (1 - p)."""
    p = case["p"]
    if p == 0.0:
        return None
    kept = _words(state["x"].numel(), state["seed"], 3) >= round(p * 2.0 ** 32)
    return kept.view(state["x"].shape).float() * (1.0 / (1.0 - p))


def _plain_dropout(case, state):
    dtype = state["x"].dtype
    factor = _factor(case, state)
    out = state["x"].float() * factor
    grad_x = (state["grad"].float() * factor).to(dtype)
    if not case["residual"]:
        return [out.to(dtype), grad_x]
    return [(out + state["residual"].float()).to(dtype), grad_x, state["grad"]]


def _norm(x, kind):
    """x without its mean (layer) over its deviation, and one over the deviation."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _norm_grad(u, h, rstd, kind):
    """x's gradient from `u` of the unit row h."""
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    return rstd * (u - h * (u * h).mean(-1, keepdim=True))


def _plain_block(case, state):
    dtype = state["x"].dtype
    t = {name: value.float() for name, value in state.items()
         if isinstance(value, torch.Tensor)}
    post, factor = case["post"], _factor(case, state)
    y = t["x"]
    if post != "none":
        unit, rstd = _norm(y, post)
        y = unit * t["post_weight"]
        if post == "layer":
            y = y + t["post_bias"]
    dropped = y if factor is None else y * factor
    gated = dropped * t["gate"] if case["gate"] else dropped
    stream = case["scale"] * t["residual"] + gated
    h, rstd_out = _norm(stream, case["norm"])
    out = h * t["weight"]
    if case["norm"] == "layer":
        out = out + t["bias"]
    outs = [out.to(dtype), stream.to(dtype)]
    if case["mode"] != "train":
        return outs
    grad = t["grad"]
    ds = t["grad_stream"] + _norm_grad(grad * t["weight"], h, rstd_out, case["norm"])
    dy = ds * t["gate"] if case["gate"] else ds
    if factor is not None:
        dy = dy * factor
    dx = dy if post == "none" else _norm_grad(dy * t["post_weight"], unit, rstd, post)
    grads = [dx, case["scale"] * ds, (grad * h).sum(0)]
    if case["norm"] == "layer":
        grads.append(grad.sum(0))
    if post != "none":
        grads.append((dy * unit).sum(0))
    if post == "layer":
        grads.append(dy.sum(0))
    if case["gate"]:
        grads.append((ds * dropped).sum(0))
    return outs + [g.to(dtype) for g in grads]


def _plain_int8(case, state):
    x = state["x"].float()
    scale = torch.clamp_min(x.abs().amax(-1, keepdim=True) / 127.0, 2.0 ** -126)
    codes = torch.round(x / scale)
    # sums past 2^24 are no float32 numbers
    wide = torch.float64 if case["in"] * 127 * 127 > 2 ** 24 else torch.float32
    sums = codes.to(wide) @ state["weight"].to(wide).t()
    z = sums.float() * scale * state["scale"] + state["bias"].float()
    if case["activation"] == "relu":
        z = torch.clamp_min(z, 0.0)
    elif case["activation"] == "gelu":
        z = z * (0.5 * torch.erfc(z * -math.sqrt(0.5)))
    if case["residual"]:
        z = z + state["residual"].float()
    return [z.to(state["x"].dtype)]


# ------------------------------------------------------------- 64 bits ---


def exact(case, seed):
    tensors = {name: value.double() for name, value in _inputs(case, seed).items()}
    return {"gated": _exact_gated, "dropout": _exact_dropout, "block": _exact_block,
            "int8": _exact_int8}[case["op"]](case, tensors, 77003 * seed + 12345)


def _exact_gated(case, t, _):
    gate_w, up_w = t["weight"].chunk(2)
    gate_b, up_b = t["bias"].chunk(2)
    a, u = torch.addmm(gate_b, t["x"], gate_w.t()), torch.addmm(up_b, t["x"], up_w.t())
    if case["activation"] == "gelu":
        phi = torch.special.ndtr(a)
        h, slope = a * phi, phi + a * torch.exp(a.square() / -2) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(a)
        rise = s * torch.sigmoid(-a)
        h, slope = (s, rise) if case["activation"] == "sigmoid" else (a * s, s + a * rise)
    outs = [h * u]
    if case["mode"] == "train":
        da, du = t["grad"] * slope * u, t["grad"] * h
        outs += [torch.addmm(da @ gate_w, du, up_w),
                 torch.cat((da.t() @ t["x"], du.t() @ t["x"])), torch.cat((da.sum(0), du.sum(0)))]
    return outs


def _multiply_halves(a, m):
    """Upper and lower 32 bits of a (32 bits) times m, from products of 16 bits."""
    lo = (a & 0xFFFF) * m
    hi = (a >> 16) * m + (lo >> 16)
    return hi >> 16, (hi & 0xFFFF) << 16 | lo & 0xFFFF


def _exact_kept(case, rows, seed):
    count = rows * case["in"]
    block = torch.arange(-(-count // 4), device=DEVICE)
    x = [block % 2 ** 32, block // 2 ** 32, torch.full_like(block, 3), torch.zeros_like(block)]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for turn in range(10):
        k = [(key[0] + turn * 0x9E3779B9) % 2 ** 32, (key[1] + turn * 0xBB67AE85) % 2 ** 32]
        upper0, lower0 = _multiply_halves(x[0], 0xD2511F53)
        upper1, lower1 = _multiply_halves(x[2], 0xCD9E8D57)
        x = [upper1.bitwise_xor(x[1]).bitwise_xor(k[0]), lower1,
             upper0.bitwise_xor(x[3]).bitwise_xor(k[1]), lower0]
    unit = torch.stack(x, 1).flatten()[:count].double() / 2.0 ** 32
    return (unit >= round(case["p"] * 2.0 ** 32) / 2.0 ** 32).view(rows, -1)


def _exact_dropout(case, t, seed):
    drop = ~_exact_kept(case, case["rows"], seed)
    keep = 1.0 - case["p"]
    out, grad = (v.masked_fill(drop, 0.0) / keep for v in (t["x"], t["grad"]))
    return [out + t["residual"], grad, t["grad"]] if case["residual"] else [out, grad]


def _exact_norm(x, kind):
    centre = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else 0.0
    sigma = ((x - centre).square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    return (x - centre) / sigma, sigma


def _exact_norm_grad(g, unit, sigma, kind):
    n = unit.shape[-1]
    along = (g * unit).sum(-1, keepdim=True) / n
    level = g.sum(-1, keepdim=True) / n if kind == "layer" else 0.0
    return (g - level - unit * along) / sigma


def _exact_block(case, t, seed):
    one = torch.ones((), dtype=torch.float64, device=DEVICE)
    gate, post = t.get("gate", one), case["post"]
    weight = one
    if case["p"]:
        weight = _exact_kept(case, case["rows"], seed).double() / (1.0 - case["p"])
    y = t["x"]
    if post != "none":
        inner, inner_sigma = _exact_norm(y, post)
        y = torch.addcmul(t.get("post_bias", one * 0.0), inner, t["post_weight"])
    stream = torch.addcmul(t["residual"] * case["scale"], y * weight, gate)
    unit, sigma = _exact_norm(stream, case["norm"])
    outs = [torch.addcmul(t.get("bias", one * 0.0), unit, t["weight"]), stream]
    if case["mode"] != "train":
        return outs
    grad = t["grad"]
    ds = t["grad_stream"] + _exact_norm_grad(grad * t["weight"], unit, sigma, case["norm"])
    dy = ds * gate * weight
    dx = dy
    if post != "none":
        dx = _exact_norm_grad(dy * t["post_weight"], inner, inner_sigma, post)
    outs += [dx, ds * case["scale"], (grad * unit).sum(0)]
    if case["norm"] == "layer":
        outs.append(grad.sum(0))
    if post != "none":
        outs.append((dy * inner).sum(0))
    if post == "layer":
        outs.append(dy.sum(0))
    if case["gate"]:
        outs.append((ds * y * weight).sum(0))
    return outs


def _exact_int8(case, t, _):
    # the scale is a float32 number by definition, the codes go by it
    scale = (t["x"].abs().amax(-1, keepdim=True) / 127).clamp_min(2.0 ** -126).float().double()
    q = (t["x"] / scale).round()
    z = torch.addmm(t["bias"], q * scale, (t["weight"] * t["scale"][:, None]).t())
    if case["activation"] == "relu":
        z = z.clamp_min(0.0)
    elif case["activation"] == "gelu":
        z = z * torch.special.ndtr(z)
    return [z + t["residual"] if case["residual"] else z]
