"""dropout and residual_norm on the CPU: the PyTorch path against float64, their generator
against published words, and the refusals of the operators, the host module and the C-ABI."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import dropout, get_last_dispatch_report, residual_norm
from muspace_amd.runtime.layer_host import load_layer_host
from oracle import block_torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
VECTORS = ("weight", "bias", "gate", "post_weight", "post_bias")


def draw(gen, *shape, dtype=torch.float32, centre=0.0):
    return (centre + torch.randn(shape, generator=gen)).to(dtype)


# --------------------------------------------------------------- generator ---


@pytest.mark.parametrize(
    ("counter", "offset", "seed", "words"),
    [
        # the published test vectors of Philox4x32-10
        (0, 0, 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
        (2**64 - 1, 2**64 - 1, 2**64 - 1, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
        (0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822,
         "d16cfe09 94fdcceb 5001e420 24126ea1"),
    ],
)
def test_generator_against_published_words(counter, offset, seed, words):
    assert [f"{w:08x}" for w in block_torch.philox(counter, offset, seed)] == words.split()


@pytest.mark.parametrize("seed", [0, 1, 2**31, 2**63 - 1, 2**63, 2**64 - 1])
@pytest.mark.parametrize("offset", [0, 7, 2**32 + 5, 2**64 - 1])
def test_masks(seed, offset):
    for p in (0.1, 0.5, 1 - 2.0**-20):
        out = dropout(torch.ones(203), p, seed=seed, offset=offset)
        assert torch.equal(out != 0, block_torch.kept(0, 203, p, seed, offset))
    if seed < 2**63:
        tensor = torch.tensor([seed])
        assert torch.equal(dropout(torch.ones(203), 0.4, seed=tensor, offset=offset),
                           dropout(torch.ones(203), 0.4, seed=seed, offset=offset))


def test_masks_are_of_the_row_major_order():
    x = torch.ones(6, 7, 5)
    flat = dropout(x.view(-1), 0.3, seed=5)
    assert torch.equal(dropout(x, 0.3, seed=5).view(-1), flat)
    assert torch.equal(dropout(x.permute(2, 0, 1).contiguous().permute(1, 2, 0), 0.3, seed=5),
                       flat.view(6, 7, 5))


def test_share_of_kept_elements():
    """Over 2^20 elements the share errs by under 5 of its standard deviations, and pairs
    of neighbours, seeds and offsets are as if drawn apart."""
    n = 1 << 20
    for p in (0.1, 0.5):
        a = dropout(torch.ones(n), p, seed=3) != 0
        others = (dropout(torch.ones(n), p, seed=4) != 0, a.roll(1), a.roll(4),
                  dropout(torch.ones(n), p, seed=3, offset=1) != 0)
        q = 1 - p
        assert abs(a.double().mean().item() - q) < 5 * math.sqrt(q * p / n)
        for b in others:
            both = (a & b).double().mean().item()
            assert abs(both - q * q) < 5 * math.sqrt(q * q * (1 - q * q) / n)


# ------------------------------------------------------------ PyTorch path ---


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
def test_dropout_on_the_cpu(p, residual, dtype):
    gen = torch.Generator().manual_seed(0)
    x, r, g = (draw(gen, 9, 13, dtype=dtype) for _ in range(3))
    x[0, 0], x[1, 1] = math.inf, math.nan
    xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
    out = dropout(xs, p, seed=11, offset=2, residual=rs if residual else None)
    assert get_last_dispatch_report().operator == "dropout"
    assert out.dtype == dtype
    keep = block_torch.kept(0, 9 * 13, p, 11, 2).view(9, 13)
    want, bound = block_torch.dropout(x, keep, p, r if residual else None)
    finite = want.isfinite()
    assert torch.equal(finite, out.isfinite())
    assert ((out.double() - want)[finite].abs() <= bound[finite]).all()
    grads = torch.autograd.grad(out, [xs, rs] if residual else [xs], g)
    want, bound = block_torch.dropout(g, keep, p)
    assert ((grads[0].double() - want).abs() <= bound).all()
    assert not residual or torch.equal(grads[1], g)


def block_call(dtype=torch.float32, rows=7, cols=20, seed=0, wdtype=None):
    gen = torch.Generator().manual_seed(seed)
    t = {"block": draw(gen, rows, cols, dtype=dtype),
         "residual": draw(gen, rows, cols, dtype=dtype, centre=0.3)}
    for name in VECTORS:
        centre = 0.0 if name.endswith("bias") else 1.0
        t[name] = (centre + 0.3 * torch.randn(cols, generator=gen)).to(wdtype or dtype)
    return t, draw(gen, rows, cols, dtype=dtype), draw(gen, rows, cols, dtype=dtype)


def check_block(t, g, gs, p=0.0, seed=5, **kwargs):
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    normed, stream = residual_norm(**leaves, dropout_p=p, seed=seed, offset=1, **kwargs)
    keep = block_torch.kept(0, t["block"].numel(), p, seed, 1).view(t["block"].shape)
    want = block_torch.residual_norm(**t, p=p, keep=keep, grad=g, grad_stream=gs, **kwargs)
    outs = [o for o, d in ((normed, g), (stream, gs)) if d is not None]
    grads = torch.autograd.grad(outs, list(leaves.values()), [d for d in (g, gs) if d is not None],
                                allow_unused=g is None)
    got = {"normed": normed.detach(), "stream": stream.detach(), **dict(zip(leaves, grads))}
    for name, (value, bound) in want.items():
        assert got[name].shape == value.shape, name
        worst = ((got[name].double() - value).abs() / bound.clamp_min(1e-300)).max()
        assert worst <= 1, (name, float(worst))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
def test_residual_norm_on_the_cpu(post, norm, dtype):
    t, g, gs = block_call(dtype)
    if post is None:
        t = {k: v for k, v in t.items() if not k.startswith("post")}
    check_block(t, g, gs, norm=norm, post_norm=post)
    check_block(t, g, gs, p=0.3, norm=norm, post_norm=post, residual_scale=1.7)
    check_block({k: t[k] for k in ("block", "residual")}, g, gs, norm=norm, post_norm=post)
    assert get_last_dispatch_report().operator == "residual_norm"


def test_residual_norm_is_the_composition():
    t, _, _ = block_call()
    normed, stream = residual_norm(t["block"], t["residual"], t["weight"], t["bias"])
    assert torch.equal(stream, t["block"] + t["residual"])
    assert torch.equal(normed, F.layer_norm(stream, (20,), t["weight"], t["bias"]))
    assert torch.equal(residual_norm(t["block"], t["residual"], t["weight"], t["bias"],
                                     return_stream=False), normed)


def test_oracle_against_autograd():
    t, g, gs = block_call()
    t = {k: v.double() for k, v in t.items()}
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    keep = block_torch.kept(0, 140, 0.3, 1, 0).view(7, 20)
    for norm in ("layer", "rms"):
        for post in ("layer", "rms"):
            def unit(x, kind):
                c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
                return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt()

            y = unit(leaves["block"], post) * leaves["post_weight"] + leaves["post_bias"]
            stream = 0.7 * leaves["residual"] + leaves["gate"] * (y * keep / 0.7)
            normed = unit(stream, norm) * leaves["weight"] + leaves["bias"]
            grads = torch.autograd.grad([normed, stream], list(leaves.values()),
                                        [g.double(), gs.double()])
            want = block_torch.residual_norm(**t, norm=norm, post_norm=post, residual_scale=0.7,
                                             p=0.3, keep=keep, grad=g.double(),
                                             grad_stream=gs.double())
            got = {"normed": normed, "stream": stream, **dict(zip(leaves, grads))}
            for name, value in got.items():
                torch.testing.assert_close(value.detach(), want[name][0], rtol=1e-11, atol=1e-11)


def test_oracle_bounds_catch_planted_mistakes():
    """A missing correction of the projection, a gate on the wrong side of the dropout's
    scale or eps left out fall outside."""
    t, g, gs = block_call(torch.bfloat16, rows=40, cols=64)
    keep = torch.ones(40, 64, dtype=torch.bool)
    kwargs = {"norm": "layer", "post_norm": "rms", "p": 0.1, "keep": keep, "grad": g,
              "grad_stream": gs}
    want = block_torch.residual_norm(**t, **kwargs)
    for change, names in (({"norm": "rms"}, ("normed", "block")), ({"eps": 0.05}, ("normed", "stream")),
                          ({"p": 0.11}, ("stream", "block", "gate")),
                          ({"post_norm": "layer"}, ("stream", "block")),
                          ({"residual_scale": 1.02}, ("stream", "residual"))):
        wrong = block_torch.residual_norm(**t, **{**kwargs, **change})
        for name in names:
            value, bound = want[name]
            assert ((wrong[name][0] - value).abs() > bound).any(), (change, name)


# ---------------------------------------------------------------- refusals ---


@pytest.mark.parametrize(
    ("change", "error", "message"),
    [
        ({"input": torch.zeros(3, 4, dtype=torch.float64)}, TypeError, "input must be"),
        ({"p": -0.1}, ValueError, "probability"),
        ({"p": 1.5}, ValueError, "probability"),
        ({"p": math.nan}, ValueError, "probability"),
        ({"seed": None}, ValueError, "seed must be"),
        ({"seed": -1}, ValueError, "seed must be"),
        ({"seed": 1 << 64}, ValueError, "seed must be"),
        ({"seed": 0.5}, ValueError, "seed must be"),
        ({"seed": torch.zeros(2, dtype=torch.int64)}, TypeError, "seed tensor"),
        ({"seed": torch.zeros(1, dtype=torch.int32)}, TypeError, "seed tensor"),
        ({"offset": -1}, ValueError, "offset must be"),
        ({"offset": 1 << 64}, ValueError, "offset must be"),
        ({"residual": torch.zeros(4)}, ValueError, "residual must have"),
        ({"residual": torch.zeros(3, 4, dtype=torch.float16)}, TypeError, "residual must be"),
        ({"backend": "cuda"}, RuntimeError, "unknown backend"),
        ({"backend": "hip"}, RuntimeError, "requires a ROCm tensor"),
    ],
)
def test_dropout_refuses(change, error, message):
    args = {"input": torch.zeros(3, 4), "p": 0.5, "seed": 1, **change}
    with pytest.raises(error, match=message):
        dropout(args.pop("input"), args.pop("p"), **args)


@pytest.mark.parametrize(
    ("change", "error", "message"),
    [
        ({"block": torch.zeros(7, 20, dtype=torch.float64)}, TypeError, "block must be"),
        ({"block": torch.zeros(()), "residual": torch.zeros(())}, ValueError, "at least one"),
        ({"residual": torch.zeros(20)}, ValueError, "residual must have"),
        ({"residual": torch.zeros(7, 20, dtype=torch.float16)}, TypeError, "residual must be"),
        ({"norm": "batch"}, ValueError, "norm must be"),
        ({"norm": None}, ValueError, "norm must be"),
        ({"post_norm": "batch"}, ValueError, "post_norm must be"),
        ({"post_norm": None}, ValueError, "without a post_norm"),
        ({"eps": -1.0}, ValueError, "eps"),
        ({"eps": math.nan}, ValueError, "eps"),
        ({"residual_scale": math.inf}, ValueError, "residual_scale"),
        ({"residual_scale": 1e300}, ValueError, "residual_scale"),
        ({"residual_scale": math.nan}, ValueError, "residual_scale"),
        ({"dropout_p": 2.0}, ValueError, "probability"),
        ({"dropout_p": 0.1, "seed": None}, ValueError, "seed must be"),
        ({"seed": torch.zeros(1)}, TypeError, "seed tensor"),
        *[({name: torch.zeros(21)}, ValueError, f"{name} must be") for name in VECTORS],
        *[({name: torch.zeros(20, dtype=torch.float16)}, TypeError, f"{name} must be")
          for name in VECTORS],
        ({"backend": "cuda"}, RuntimeError, "unknown backend"),
        ({"backend": "hip"}, RuntimeError, "requires a ROCm tensor"),
    ],
)
def test_residual_norm_refuses(change, error, message):
    t, _, _ = block_call()
    with pytest.raises(error, match=message):
        residual_norm(**{**t, "post_norm": "layer", **change})


def test_residual_norm_refuses_vectors_of_two_types():
    t, _, _ = block_call(torch.float16)
    t["gate"] = t["gate"].float()
    with pytest.raises(TypeError, match="of one type"):
        residual_norm(**t, post_norm="layer")


@pytest.mark.parametrize("operator", ["dropout", "residual_norm"])
def test_host_refuses_tracing_and_forward_mode(operator):
    host = load_layer_host()
    r = torch.ones(3, 8)
    call = {"dropout": lambda x: host.dropout(x, r, 0.1, None, 1, 0),
            "residual_norm": lambda x: host.residual_norm(
                x, r, None, None, None, None, None, 0, -1, 1e-5, 1.0, 0.0, None, 0, 0, True)[0]}[operator]
    for graph in (False, True):
        x = torch.randn(3, 8, requires_grad=graph)
        for trace in (lambda: torch.jit.trace(call, (x,)), lambda: make_fx(call)(x.detach())):
            with pytest.raises(RuntimeError, match=f"{operator}: HIP kernels cannot be traced"):
                trace()
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones(3, 8))
            with pytest.raises(RuntimeError, match=f"{operator}: the HIP path has no forward-mode"):
                call(dual)


@pytest.mark.parametrize("shape", [(0, 5), (3, 0), (0,), (2, 0, 4)])
def test_empty_calls(shape):
    x = torch.ones(shape, requires_grad=True)
    w = torch.ones(shape[-1], requires_grad=True)
    assert dropout(x, 0.5, seed=1).shape == shape
    normed, stream = residual_norm(x, x, w, dropout_p=0.5, seed=1)
    assert normed.shape == stream.shape == shape
    dx, dw = torch.autograd.grad([normed, stream], [x, w], [normed, stream])
    assert dx.shape == shape and not dw.any()


# ------------------------------------------------------------------- C-ABI ---

# pointers are stand-ins: every call must return before anything reads them
FAR = 1 << 12


@pytest.mark.parametrize(
    ("overrides", "message"),
    [
        ({"dtype": 3}, "float32, float16 or bfloat16"),
        ({"p": -1.0}, "probability"),
        ({"p": math.nan}, "probability"),
        ({"device_seed": FAR + 4}, "8-byte aligned"),
        ({"count": -1}, "invalid count"),
        ({"x": None}, "null tensor pointer"),
        ({"output": None}, "null tensor pointer"),
    ],
)
def test_dropout_abi_refuses(native_lib, overrides, message):
    args = dict(x=FAR, dtype=0, residual=None, output=FAR, count=8, p=0.5, seed=1,
                device_seed=None, offset=0, stream=None)
    args.update(overrides)
    assert native_lib.raw("dropout_forward")(*args.values()) == 1
    assert message in native_lib.last_error()


def test_dropout_abi_empty_is_a_no_op(native_lib):
    assert native_lib.raw("dropout_forward")(None, 0, None, None, 0, 0.5, 1, None, 0, None) == 0


def forward_args(**overrides):
    args = dict(block=FAR, dtype=2, residual=FAR, weight=None, bias=None, gate=None,
                post_weight=None, post_bias=None, weight_dtype=0, output=FAR, stream_values=None,
                stats=None, post_stats=None, rows=4, cols=8, norm=0, post_norm=-1, eps=1e-5,
                scale=1.0, p=0.0, seed=0, device_seed=None, offset=0, stream=None)
    args.update(overrides)
    return list(args.values())


@pytest.mark.parametrize(
    ("overrides", "code", "message"),
    [
        ({"dtype": 5}, 1, "float32, float16 or bfloat16"),
        ({"weight_dtype": 1}, 1, "weights must be"),
        ({"rows": -1}, 1, "invalid dims"),
        ({"norm": 2}, 1, "norm must be"),
        ({"norm": -1}, 1, "norm must be"),
        ({"post_norm": 2}, 1, "post_norm must be"),
        ({"cols": 1 << 21}, 2, "32-bit"),
        ({"rows": 1 << 31}, 2, "32-bit"),
        ({"p": 2.0}, 1, "probability"),
        ({"block": None}, 1, "null tensor pointer"),
        ({"residual": None}, 1, "null tensor pointer"),
        ({"output": None}, 1, "null tensor pointer"),
        ({"stats": FAR + 8}, 1, "16-byte aligned"),
    ],
)
def test_residual_norm_forward_abi_refuses(native_lib, overrides, code, message):
    assert native_lib.raw("residual_norm_forward")(*forward_args(**overrides)) == code
    assert message in native_lib.last_error()


def backward_args(**overrides):
    args = dict(grad=FAR, grad_stream=FAR, dtype=2, block=FAR, residual=FAR, stream_values=FAR,
                weight=None, gate=None, post_weight=None, post_bias=None, weight_dtype=0, stats=FAR,
                post_stats=FAR, grad_block=FAR, grad_residual=FAR, grad_weight=FAR, grad_bias=None,
                grad_gate=None, grad_post_weight=None, grad_post_bias=None, rows=4, cols=8, norm=0,
                post_norm=-1, scale=1.0, p=0.0, seed=0, device_seed=None, offset=0, workspace=FAR,
                nbytes=1 << 20, stream=None)
    args.update(overrides)
    return list(args.values())


@pytest.mark.parametrize(
    ("overrides", "code", "message"),
    [
        ({"dtype": -1}, 1, "float32, float16 or bfloat16"),
        ({"cols": -1}, 1, "invalid dims"),
        ({"cols": 1 << 21}, 2, "32-bit"),
        ({"p": -0.5}, 1, "probability"),
        ({"residual": None}, 1, "null tensor pointer"),
        ({"block": None}, 1, "null tensor pointer"),
        ({"dtype": 0, "stream_values": None}, 1, "null tensor pointer"),
        ({"stats": None}, 1, "null tensor pointer"),
        ({"stats": FAR + 8}, 1, "16-byte aligned"),
        ({"dtype": 0, "grad_gate": FAR, "block": None}, 1, "null tensor pointer"),
        ({"post_norm": 0, "post_stats": None}, 1, "null tensor pointer"),
        ({"grad_post_weight": FAR}, 1, "without one"),
        ({"workspace": None}, 1, "workspace"),
        ({"workspace": FAR + 4}, 1, "workspace"),
        ({"nbytes": 8}, 1, "workspace"),
    ],
)
def test_residual_norm_backward_abi_refuses(native_lib, overrides, code, message):
    assert native_lib.raw("residual_norm_backward")(*backward_args(**overrides)) == code
    assert message in native_lib.last_error()


def test_residual_norm_abi_without_work_is_a_no_op(native_lib):
    assert native_lib.raw("residual_norm_forward")(*forward_args(rows=0, block=None)) == 0
    none = dict(grad_block=None, grad_residual=None, grad_weight=None)
    assert native_lib.raw("residual_norm_backward")(*backward_args(**none)) == 0
    size = native_lib.raw("residual_norm_backward_workspace_size")
    assert size(2, 100, 64, 0) == size(7, 100, 64, 2) == 0
    # 8 pieces a row: 16 lanes, 16 rows a workgroup, 7 workgroups
    assert size(2, 100, 64, 3) == 7 * 3 * 64 * 4
