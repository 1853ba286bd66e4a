"""linear, its 8-bit checkpoint and layer_norm on the CPU: the PyTorch path, the
refusals of the operators and of the C-ABI, and the pins of their oracle."""

import math

import pytest
import torch
import torch.nn.functional as F

from muspace_amd import (
    checkpoint_int8,
    checkpoint_restore,
    get_last_dispatch_report,
    layer_norm,
    linear,
)
from oracle import dense_torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(rows=7, inner=40, outer=12, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def draw(*shape):
        return torch.randn(shape, generator=gen).to(dtype)

    return draw(rows, inner), draw(outer, inner), draw(outer), draw(rows, outer), draw(rows, outer)


# ------------------------------------------------------------ PyTorch path ---


@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
def test_linear_on_the_cpu_is_the_composition(activation):
    x, w, b, r, g = inputs()
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    out = linear(*leaves[:3], activation=activation, residual=leaves[3])
    assert get_last_dispatch_report().operator == "linear"
    assert get_last_dispatch_report().selected_backend == "reference"
    act = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu}[activation]
    assert torch.equal(out, act(F.linear(x, w, b)) + r)
    grads = torch.autograd.grad(out, leaves, g)
    results, bounds = dense_torch.linear(x, w, b, activation, r, g)
    for a, e, t in zip([out, *grads[:3]], results, bounds):
        assert ((a.double() - e).abs() <= t).all()
    assert torch.equal(grads[3], g)


@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
def test_checkpoint_on_the_cpu_changes_the_weight_gradient_only(activation):
    x, w, b, r, g = inputs(rows=30, inner=70)
    plain = [t.clone().requires_grad_() for t in (x, w, b, r)]
    kept = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want_out = linear(*plain[:3], activation=activation, residual=plain[3])
    out = linear(*kept[:3], activation=activation, residual=kept[3], checkpoint="int8")
    torch.testing.assert_close(out, want_out, rtol=1e-5, atol=1e-5)
    want = torch.autograd.grad(want_out, plain, g)
    got = torch.autograd.grad(out, kept, g)
    for i in (0, 2, 3):
        torch.testing.assert_close(got[i], want[i], rtol=1e-5, atol=1e-5)
    restored = dense_torch.checkpoint(x)[2]
    results, bounds = dense_torch.linear(x, w, b, activation, r, g, restored)
    assert ((got[1].double() - results[2]).abs() <= bounds[2]).all()
    assert not torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 31, 32, 33, 100])
def test_checkpoint_codes(cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    info = torch.finfo(dtype)
    x = torch.randn((40, cols), generator=gen)
    x *= torch.exp2(torch.randint(-40, 12, (40, 1), generator=gen).float())
    x = x.to(dtype)
    x[0], x[1], x[2], x[3] = 0.0, info.max, -info.max, info.smallest_normal
    x[4] = info.smallest_normal / 4
    x[5, 0], x[6, cols - 1] = math.inf, math.nan
    x[7], x[8], x[9] = 127.0, 127.5, -63.5
    codes, scales = checkpoint_int8(x)
    e_codes, e_scales, e_values = dense_torch.checkpoint(x)
    assert torch.equal(codes, e_codes) and torch.equal(scales, e_scales)
    assert codes.shape == (40, (cols + 31) // 32 * 32) and codes.dtype == torch.int8
    restored = checkpoint_restore(codes, scales, cols, dtype)
    assert restored.dtype == dtype
    assert torch.equal(torch.nan_to_num(restored.double(), nan=-1.0),
                       torch.nan_to_num(e_values, nan=-1.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_error_is_half_a_step(dtype):
    x = inputs(rows=50, inner=96, dtype=dtype)[0]
    codes, scales = checkpoint_int8(x)
    restored = checkpoint_restore(codes, scales, 96, dtype).double()
    step = torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)
    assert ((restored - x.double()).abs() <= step / 2).all()
    # the step is the smallest: half of it would not reach the block's largest
    top = x.double().abs().view(50, 3, 32).amax(-1).repeat_interleave(32, dim=1)
    assert (127 * step >= top).all() and (127 * step / 2 < top).all()


def test_checkpoint_flattens_leading_dimensions():
    x = inputs(rows=12, inner=33)[0]
    codes, scales = checkpoint_int8(x.view(3, 4, 33))
    want = checkpoint_int8(x)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_on_the_cpu(dtype):
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn((9, 50), generator=gen) + 1).to(dtype)
    w = torch.randn(50, generator=gen).to(dtype)
    b = torch.randn(50, generator=gen).to(dtype)
    out = layer_norm(x, w, b)
    assert get_last_dispatch_report().operator == "layer_norm"
    assert torch.equal(out, F.layer_norm(x, (50,), w, b))
    assert torch.equal(layer_norm(x), F.layer_norm(x, (50,)))
    mixed = layer_norm(x, w.float(), b.float())
    assert mixed.dtype == dtype
    assert torch.equal(mixed, F.layer_norm(x.float(), (50,), w.float(), b.float()).to(dtype))


# ---------------------------------------------------------------- refusals ---


@pytest.mark.parametrize(
    ("change", "error", "message"),
    [
        ({"input": torch.zeros(3, 40, dtype=torch.float64)}, TypeError, "input must be"),
        ({"input": torch.zeros((), dtype=torch.float32)}, ValueError, "at least one dimension"),
        ({"weight": torch.zeros(12, 41)}, ValueError, "weight must be"),
        ({"weight": torch.zeros(40)}, ValueError, "weight must be"),
        ({"weight": torch.zeros(12, 40, dtype=torch.float16)}, TypeError, "weight must be"),
        ({"bias": torch.zeros(11)}, ValueError, "bias must be"),
        ({"bias": torch.zeros(12, dtype=torch.bfloat16)}, TypeError, "bias must be"),
        ({"residual": torch.zeros(12)}, ValueError, "residual must have"),
        ({"residual": torch.zeros(7, 12, dtype=torch.float16)}, TypeError, "residual must be"),
        ({"activation": "silu"}, ValueError, "activation must be"),
        ({"checkpoint": "fp8"}, ValueError, "checkpoint must be"),
        ({"backend": "cuda"}, RuntimeError, "unknown backend"),
        ({"backend": "hip"}, RuntimeError, "requires a ROCm tensor"),
    ],
)
def test_linear_refuses(change, error, message):
    x, w, b, r, _ = inputs()
    args = {"input": x, "weight": w, "bias": b, "residual": r, **change}
    with pytest.raises(error, match=message):
        linear(args.pop("input"), args.pop("weight"), args.pop("bias"), **args)


@pytest.mark.parametrize(
    ("args", "kwargs", "error", "message"),
    [
        ((torch.zeros(2, 4, dtype=torch.float64),), {}, TypeError, "input must be"),
        ((torch.zeros(()),), {}, ValueError, "at least one dimension"),
        ((torch.zeros(2, 4), torch.ones(3)), {}, ValueError, "weight must be"),
        ((torch.zeros(2, 4), torch.ones(4, dtype=torch.float16)), {}, TypeError, "weight must be"),
        ((torch.zeros(2, 4), torch.ones(4), torch.ones(2, 4)), {}, ValueError, "bias must be"),
        ((torch.zeros(2, 4, dtype=torch.float16), torch.ones(4),
          torch.ones(4, dtype=torch.float16)), {}, TypeError, "of one type"),
        ((torch.zeros(2, 4),), {"eps": -1.0}, ValueError, "eps"),
        ((torch.zeros(2, 4),), {"eps": math.nan}, ValueError, "eps"),
        ((torch.zeros(2, 4),), {"backend": "hip"}, RuntimeError, "requires a ROCm tensor"),
    ],
)
def test_layer_norm_refuses(args, kwargs, error, message):
    with pytest.raises(error, match=message):
        layer_norm(*args, **kwargs)


def test_checkpoint_refuses():
    with pytest.raises(TypeError, match="input must be"):
        checkpoint_int8(torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one dimension"):
        checkpoint_int8(torch.zeros(()))


# ------------------------------------------------------------------- C-ABI ---

# pointers are stand-ins: every call must return before anything reads them
FAR = 1 << 12


def forward_args(**overrides):
    args = dict(x=FAR, dtype=0, weight=FAR, bias=None, residual=None, output=FAR, mask=None,
                z=None, codes=None, scales=None, rows=4, inner=8, outer=8, activation=0, stream=None)
    args.update(overrides)
    return list(args.values())


@pytest.mark.parametrize(
    ("overrides", "code", "message"),
    [
        ({"dtype": 3}, 1, "float32, float16 or bfloat16"),
        ({"dtype": -1}, 1, "float32, float16 or bfloat16"),
        ({"rows": -1}, 1, "invalid dims"),
        ({"outer": -4}, 1, "invalid dims"),
        ({"activation": 3}, 1, "activation must be"),
        ({"rows": 1 << 31}, 2, "32-bit"),
        ({"inner": (1 << 20) + 1}, 2, "32-bit"),
        ({"rows": 1 << 30, "outer": 1 << 20}, 2, "32-bit"),
        ({"rows": (1 << 31) - 300, "inner": 200}, 2, "32-bit"),
        ({"inner": 1 << 20, "outer": 1 << 20}, 2, "32-bit"),
        ({"x": None}, 1, "null tensor pointer"),
        ({"weight": None}, 1, "null tensor pointer"),
        ({"output": None}, 1, "null tensor pointer"),
        ({"codes": FAR}, 1, "codes and scales come together"),
        ({"scales": FAR}, 1, "codes and scales come together"),
        ({"codes": FAR + 2, "scales": FAR}, 1, "8-byte aligned"),
    ],
)
def test_linear_forward_abi_refuses(native_lib, overrides, code, message):
    assert native_lib.raw("linear_forward")(*forward_args(**overrides)) == code
    assert message in native_lib.last_error()


def test_linear_forward_abi_empty_is_a_no_op(native_lib):
    for overrides in ({"rows": 0}, {"outer": 0}):
        args = forward_args(x=None, weight=None, output=None, **overrides)
        assert native_lib.raw("linear_forward")(*args) == 0
        assert native_lib.last_error() == ""


def backward_args(**overrides):
    args = dict(grad=FAR, dtype=0, x=FAR, codes=None, scales=None, weight=FAR, mask=FAR, z=FAR,
                grad_input=FAR, grad_weight=FAR, grad_bias=FAR, rows=4, inner=8, outer=8,
                activation=0, workspace=FAR, nbytes=1 << 20, stream=None)
    args.update(overrides)
    return list(args.values())


@pytest.mark.parametrize(
    ("overrides", "message"),
    [
        ({"dtype": 9}, "float32, float16 or bfloat16"),
        ({"inner": -1}, "invalid dims"),
        ({"activation": -1}, "activation must be"),
        ({"grad": None}, "null tensor pointer"),
        ({"x": None}, "null tensor pointer"),
        ({"weight": None}, "null tensor pointer"),
        ({"codes": FAR}, "codes and scales come together"),
        ({"scales": FAR}, "codes and scales come together"),
        ({"codes": FAR + 4, "scales": FAR}, "8-byte aligned"),
        ({"activation": 1, "mask": None}, "null tensor pointer"),
        ({"activation": 2, "z": None}, "null tensor pointer"),
        ({"activation": 2, "workspace": None}, "workspace"),
        ({"activation": 2, "workspace": FAR + 16}, "workspace"),
        ({"rows": 100000, "nbytes": 256}, "workspace"),
    ],
)
def test_linear_backward_abi_refuses(native_lib, overrides, message):
    assert native_lib.raw("linear_backward")(*backward_args(**overrides)) == 1
    assert message in native_lib.last_error()


def test_linear_backward_abi_without_gradients_is_a_no_op(native_lib):
    args = backward_args(grad_input=None, grad_weight=None, grad_bias=None, grad=None)
    assert native_lib.raw("linear_backward")(*args) == 0


def test_linear_workspace(native_lib):
    size = native_lib.raw("linear_backward_workspace_size")
    assert size(9, 4, 8, 8, 0) == 0
    assert size(0, 0, 8, 8, 0) == 0
    assert size(2, 40, 8, 8, 0) == 0  # a short sum is not cut
    # gelu: dz padded to 256 bytes, in 16-bit types with what rounding left
    assert size(0, 40, 8, 8, 2) == 40 * 8 * 4
    assert size(2, 40, 8, 8, 2) == 2 * (40 * 8 * 2 + 128)
    assert 0 < size(2, 40000, 256, 512, 0) < 1 << 28


def test_checkpoint_abi_refuses(native_lib):
    fn = native_lib.raw("linear_checkpoint")
    assert fn(FAR, 5, FAR, FAR, 4, 8, None) == 1
    assert fn(FAR, 0, FAR, FAR, -4, 8, None) == 1
    assert fn(FAR, 0, FAR + 4, FAR, 4, 8, None) == 1
    assert "8-byte aligned" in native_lib.last_error()
    assert fn(FAR, 0, None, FAR, 4, 8, None) == 1
    assert "null tensor pointer" in native_lib.last_error()
    assert fn(None, 0, None, None, 0, 8, None) == 0


def norm_args(**overrides):
    args = dict(grad=FAR, dtype=2, x=FAR, weight=FAR, weight_dtype=2, stats=FAR, grad_input=FAR,
                grad_weight=FAR, grad_bias=FAR, rows=4, cols=8, workspace=FAR, nbytes=1 << 20,
                stream=None)
    args.update(overrides)
    return list(args.values())


@pytest.mark.parametrize(
    ("overrides", "code", "message"),
    [
        ({"dtype": 4}, 1, "float32, float16 or bfloat16"),
        ({"weight_dtype": 1}, 1, "weight and bias"),
        ({"cols": -1}, 1, "invalid dims"),
        ({"cols": 1 << 21}, 2, "32-bit"),
        ({"rows": 1 << 31}, 2, "32-bit"),
        ({"grad": None}, 1, "null tensor pointer"),
        ({"stats": None}, 1, "null tensor pointer"),
        ({"workspace": None}, 1, "workspace"),
        ({"workspace": FAR + 4}, 1, "workspace"),
        ({"nbytes": 8}, 1, "workspace"),
    ],
)
def test_layer_norm_abi_refuses(native_lib, overrides, code, message):
    assert native_lib.raw("layer_norm_backward")(*norm_args(**overrides)) == code
    assert message in native_lib.last_error()


def test_layer_norm_forward_abi_refuses(native_lib):
    fn = native_lib.raw("layer_norm_forward")
    assert fn(FAR, 3, None, None, 0, FAR, None, 4, 8, 1e-5, None) == 1
    assert fn(None, 0, None, None, 0, FAR, None, 4, 8, 1e-5, None) == 1
    assert "null tensor pointer" in native_lib.last_error()
    assert fn(None, 0, None, None, 0, None, None, 0, 8, 1e-5, None) == 0


def test_host_module_missing_is_an_error(monkeypatch, tmp_path):
    """A device call without the host module raises and says how to build it; CPU calls
    keep the PyTorch path."""
    from muspace_amd.ops import layer_common
    from muspace_amd.runtime import layer_host

    monkeypatch.setattr(layer_host, "module_path", lambda: tmp_path / "missing.so")
    layer_host.load_layer_host.cache_clear()
    try:
        assert "python -m muspace_amd.build" in layer_host.layer_host_error()
        with pytest.raises(RuntimeError, match="missing from this installation"):
            layer_common.require_native()
        monkeypatch.setattr(layer_common, "is_rocm_tensor", lambda t: True)
        x = torch.zeros(2, 4)
        monkeypatch.setattr("muspace_amd.runtime.kernel_dispatch.is_rocm_tensor", lambda t: True)
        with pytest.raises(RuntimeError, match="missing from this installation"):
            layer_norm(x)
        assert get_last_dispatch_report().selected_backend == "error"
    finally:
        layer_host.load_layer_host.cache_clear()
    monkeypatch.undo()
    assert torch.equal(layer_norm(torch.zeros(2, 4)), torch.zeros(2, 4))
    assert layer_host.load_layer_host() is layer_host.load_layer_host()


def test_host_module_binds_every_entry(native_lib):
    """The host module takes its entry points from the loaded library."""
    from muspace_amd.runtime import layer_host, native

    assert set(layer_host._BOUND) <= set(native._EXPORTS)
    host = layer_host.load_layer_host()
    with pytest.raises(Exception, match="linear_forward|map::at|at"):
        host.bind({"muspace_last_error": 1})
    layer_host.load_layer_host.cache_clear()  # a partial bind: load (and bind) anew
    layer_host.load_layer_host()


# ------------------------------------------------------------------ oracle ---


@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
def test_oracle_linear_against_autograd(activation):
    x, w, b, r, g = (t.double().requires_grad_() for t in inputs())
    act = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu}[activation]
    y = act(F.linear(x, w, b)) + r
    grads = torch.autograd.grad(y, [x, w, b], g.detach())
    results, _ = dense_torch.linear(x.detach().float(), w.detach().float(), b.detach().float(),
                                    activation, r.detach().float(), g.detach().float())
    for a, e in zip([y, *grads], results):
        torch.testing.assert_close(a.detach(), e, rtol=1e-12, atol=1e-12)


def test_oracle_layer_norm_against_autograd():
    gen = torch.Generator().manual_seed(3)
    x, w, b, g = (torch.randn(s, generator=gen).double().requires_grad_()
                  for s in ((6, 31), (31,), (31,), (6, 31)))
    y = F.layer_norm(x, (31,), w, b, 1e-5)
    grads = torch.autograd.grad(y, [x, w, b], g.detach())
    results, _ = dense_torch.layer_norm(x.detach().float(), w.detach().float(),
                                        b.detach().float(), 1e-5, g.detach().float())
    for a, e in zip([y, *grads], results):
        torch.testing.assert_close(a.detach(), e, rtol=1e-11, atol=1e-11)


@pytest.mark.parametrize("dtype", DTYPES)
def test_oracle_bounds_catch_planted_mistakes(dtype):
    """The bounds are tight enough: a dropped bias, a missed last k, a swapped
    activation or statistics over one column less fall outside."""
    x, w, b, r, g = inputs(dtype=dtype)
    (y, dx, dw, db), bounds = dense_torch.linear(x, w, b, "relu", r, g)
    short = dense_torch.linear(x[:, :-1], w[:, :-1], b, "relu", r)[0][0]
    for wrong in (short, dense_torch.linear(x, w, None, "relu", r)[0][0],
                  dense_torch.linear(x, w, b, "gelu", r)[0][0]):
        assert ((wrong - y).abs() > bounds[0]).any()
    fewer = dense_torch.linear(x[:-1], w, b, "relu", r[:-1], g[:-1])[0]
    assert ((fewer[2] - dw).abs() > bounds[2]).any() and ((fewer[3] - db).abs() > bounds[3]).any()
    (y, dx), bounds = (v[:2] for v in dense_torch.layer_norm(x, None, None, 1e-5, x * 0 + x.flip(0)))
    less = dense_torch.layer_norm(x[:, :-1], None, None, 1e-5)[0][0]
    assert ((less - y[:, :-1]).abs() > bounds[0][:, :-1]).any()
