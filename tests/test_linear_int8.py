"""linear_int8 and quantize_int8 on the CPU: the PyTorch path, and the refusals of the
operators, the host module and the C-ABI."""

import math

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import get_last_dispatch_report, linear_int8, quantize_int8
from muspace_amd.runtime.layer_host import load_layer_host
from oracle import dense_torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(rows=7, inner=40, outer=12, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def draw(*shape):
        return torch.randn(shape, generator=gen)

    codes, scale = quantize_int8(draw(outer, inner))
    return (draw(rows, inner).to(dtype), codes, scale, draw(outer).to(dtype),
            draw(rows, outer).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 15, 16, 17, 300])
def test_quantize(cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    info = torch.finfo(dtype)
    x = torch.randn((40, cols), generator=gen)
    x *= torch.exp2(torch.randint(-40, 12, (40, 1), generator=gen).float())
    x = x.to(dtype)
    x[0], x[1], x[2], x[3] = 0.0, info.max, -info.max, info.smallest_normal
    x[4] = info.smallest_normal / 4
    x[5, 0], x[6, cols - 1] = math.inf, math.nan
    x[7] = torch.arange(cols) % 128
    x[7, 0] = 127.0
    x[8] = torch.arange(cols) % 127 + 0.5  # ties
    x[8, 0] = -127.0
    codes, scales = quantize_int8(x)
    want, want_scales = dense_torch.quantize(x)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scales.shape == (40,)
    assert torch.equal(codes, want)
    assert torch.equal(scales.nan_to_num(-1), want_scales.nan_to_num(-1))
    keep = [i for i in range(40) if i not in (5, 6)]
    back = codes[keep].double() * scales[keep].double()[:, None]
    # half a step, and the quotient's and the scale's roundings
    limit = scales[keep].double()[:, None] * (0.5 + 127 * 2.0**-23)
    assert ((back - x[keep].double()).abs() <= limit).all()
    assert codes[keep].abs().max() <= 127
    assert torch.equal(quantize_int8(x.view(4, 10, cols))[0].view(40, cols), codes)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_int8_on_the_cpu(residual, activation, dtype):
    x, w, s, b, r = inputs(dtype=dtype)
    r = r if residual else None
    out = linear_int8(x, w, s, b, activation=activation, residual=r)
    assert get_last_dispatch_report().operator == "linear_int8"
    assert out.dtype == dtype
    y, bound = dense_torch.linear_int8(x, w, s, b, activation, r)
    assert ((out.double() - y).abs() <= bound).all()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(linear_int8(x, w, s, b, activation=activation, residual=r), out)


def test_near_the_layer_it_stands_for():
    """Errors of codes are spread evenly over a step of top / 127: the result is within 2^-6 of
    the product's root mean square (top is 3.5 deviations: 3.5 / 127 / sqrt(12) = 2^-7, twice)."""
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn((50, 512), generator=gen), torch.randn((64, 512), generator=gen)
    want = x @ w.t()
    out = linear_int8(x, *quantize_int8(w))
    assert (out - want).square().mean().sqrt() < 2.0**-6 * want.square().mean().sqrt()


def test_oracle_bounds_catch_planted_mistakes():
    x, w, s, b, r = inputs(rows=20, inner=100)
    y, bound = dense_torch.linear_int8(x, w, s, b, "gelu", r)
    one = w.clone()
    one[3, 7] += 1
    for wrong in (dense_torch.linear_int8(x, one, s, b, "gelu", r)[0],
                  dense_torch.linear_int8(x, w, s.roll(1), b, "gelu", r)[0],
                  dense_torch.linear_int8(x, w, s, b, "relu", r)[0],
                  dense_torch.linear_int8(x, w, s, None, "gelu", r)[0]):
        assert ((wrong - y).abs() > bound).any()


def test_empty_calls():
    for shape, outer in (((0, 20), 6), ((2, 0, 5), 6), ((3, 0), 6), ((3, 20), 0), ((0,), 6)):
        x = torch.ones(shape)
        w, s = quantize_int8(torch.ones(outer, shape[-1]))
        out = linear_int8(x, w, s, torch.ones(outer))
        assert out.shape == (*shape[:-1], outer)
        codes, scales = quantize_int8(x)
        assert codes.shape == shape and scales.shape == shape[:-1]
    assert torch.equal(linear_int8(torch.ones(3, 0), *quantize_int8(torch.ones(6, 0)), torch.ones(6)),
                       torch.ones(3, 6))


@pytest.mark.parametrize(
    ("change", "error", "message"),
    [
        ({"input": torch.zeros(7, 40, dtype=torch.float64)}, TypeError, "input must be"),
        ({"input": torch.zeros(())}, ValueError, "at least one dimension"),
        ({"weight": torch.zeros(12, 40)}, TypeError, "weight must be int8"),
        ({"weight": torch.zeros(12, 41, dtype=torch.int8)}, ValueError, "weight must be"),
        ({"weight": torch.zeros(40, dtype=torch.int8)}, ValueError, "weight must be"),
        ({"weight_scale": torch.ones(11)}, ValueError, "weight_scale must be"),
        ({"weight_scale": torch.ones(12).half()}, TypeError, "weight_scale must be"),
        ({"bias": torch.zeros(11)}, ValueError, "bias must be"),
        ({"bias": torch.zeros(12).half()}, TypeError, "bias must be"),
        ({"residual": torch.zeros(12)}, ValueError, "residual must have"),
        ({"residual": torch.zeros(7, 12).half()}, TypeError, "residual must be"),
        ({"activation": "silu"}, ValueError, "activation must be"),
        ({"input": torch.zeros(7, 40, requires_grad=True)}, RuntimeError, "no gradients"),
        ({"bias": torch.zeros(12, requires_grad=True)}, RuntimeError, "no gradients"),
        ({"input": torch.zeros(1, 131088), "weight": torch.zeros(12, 131088, dtype=torch.int8),
          "residual": None}, ValueError, "in_features must be at most"),
        ({"backend": "cuda"}, RuntimeError, "unknown backend"),
        ({"backend": "hip"}, RuntimeError, "requires a ROCm tensor"),
    ],
)
def test_refusals(change, error, message):
    x, w, s, b, r = inputs()
    with pytest.raises(error, match=message):
        linear_int8(**{"input": x, "weight": w, "weight_scale": s, "bias": b, "residual": r, **change})
    with torch.no_grad():
        if "no gradients" in message:
            linear_int8(**{"input": x, "weight": w, "weight_scale": s, "bias": b, **change})


def test_quantize_refuses():
    with pytest.raises(TypeError, match="input must be"):
        quantize_int8(torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one dimension"):
        quantize_int8(torch.zeros(()))


def test_host_refuses_tracing_and_gradients():
    host = load_layer_host()
    w, s = torch.ones(4, 8, dtype=torch.int8), torch.ones(4)
    x = torch.randn(3, 8)
    for name, call in (("linear_int8", lambda t: host.linear_int8(t, w, s, None, None, 0)),
                       ("quantize_int8", lambda t: host.quantize(t)[0])):
        for trace in (lambda: torch.jit.trace(call, (x,)), lambda: make_fx(call)(x)):
            with pytest.raises(RuntimeError, match=f"{name}: HIP kernels cannot be traced"):
                trace()
    with pytest.raises(RuntimeError, match="linear_int8 has no gradients"):
        host.linear_int8(x.clone().requires_grad_(), w, s, None, None, 0)


# pointers are stand-ins: every call must return before anything reads them
FAR = 1 << 12


@pytest.mark.parametrize(
    ("overrides", "code", "message"),
    [
        ({"dtype": 3}, 1, "float32, float16 or bfloat16"),
        ({"rows": -1}, 1, "invalid dims"),
        ({"outer": -4}, 1, "invalid dims"),
        ({"activation": 3}, 1, "activation must be"),
        ({"rows": 1 << 31}, 2, "32-bit"),
        ({"inner": (1 << 17) + 1}, 2, "32-bit"),
        ({"outer": (1 << 20) + 1}, 2, "32-bit"),
        ({"rows": 1 << 30, "outer": 1 << 20}, 2, "32-bit"),
        ({"x": None}, 1, "null tensor pointer"),
        ({"weight": None}, 1, "null tensor pointer"),
        ({"scales": None}, 1, "null tensor pointer"),
        ({"output": None}, 1, "null tensor pointer"),
        ({"workspace": None}, 1, "workspace"),
        ({"workspace": FAR + 16}, 1, "workspace"),
        ({"nbytes": 128}, 1, "workspace"),
    ],
)
def test_forward_abi_refuses(native_lib, overrides, code, message):
    args = dict(x=FAR, dtype=0, weight=FAR, scales=FAR, bias=None, residual=None, output=FAR,
                rows=5, inner=2064, outer=8, activation=0, workspace=FAR, nbytes=1 << 20, stream=None)
    args.update(overrides)
    assert native_lib.raw("linear_int8_forward")(*args.values()) == code
    assert message in native_lib.last_error()


def test_quantize_abi_refuses(native_lib):
    fn = native_lib.raw("quantize_int8")
    for args, code in (((FAR, 4, FAR, FAR, 4, 8), 1), ((FAR, 0, FAR, FAR, -4, 8), 1),
                       ((FAR, 0, FAR, FAR, 4, -8), 1), ((FAR, 0, FAR, FAR, 4, (1 << 20) + 1), 2),
                       ((None, 0, FAR, FAR, 4, 8), 1), ((FAR, 0, None, FAR, 4, 8), 1),
                       ((FAR, 0, FAR, None, 4, 8), 1), ((None, 0, None, None, 0, 8), 0)):
        assert fn(*args, None) == code


def test_abi_without_work_and_workspace(native_lib):
    fn = native_lib.raw("linear_int8_forward")
    assert fn(None, 0, None, None, None, None, None, 0, 8, 8, 0, None, 0, None) == 0
    assert fn(None, 0, None, None, None, None, None, 4, 8, 0, 0, None, 0, None) == 0
    size = native_lib.raw("linear_int8_workspace_size")
    assert size(7, 4, 8, 8) == size(0, 0, 8, 8) == 0
    # codes in rows of whole 16 bytes, then a scale a row
    assert size(2, 100, 2050, 8) == 206592 + 512
    # few rows and few results are quantised where they are multiplied
    assert size(2, 4, 12288, 4096) == size(2, 1, 49152, 4096) == size(2, 300, 256, 256) == 0
    assert size(2, 4, 12289, 4096) > 0 and size(2, 40000, 264, 512) > 0
    # and many short rows
    assert size(2, 40000, 256, 512) == 0 and size(2, 40000, 256, 513) > 0
    assert size(2, 24512, 256, 512) > 0 and size(2, 24513, 256, 512) == 0


def test_no_launch_holds_too_many_threads(native_lib):
    """2^32 threads are one too many: 2^24 workgroups of 256. Rows past 64 times that, less one
    workgroup, are quantised into the workspace first, as longer rows are."""
    size = native_lib.raw("linear_int8_workspace_size")
    for rows in ((1 << 30) - 64, 1 << 20):
        assert size(2, rows, 80, 16) == 0
    for rows in ((1 << 30) - 63, 1 << 30, (1 << 30) + (1 << 20), (1 << 31) - 257):
        assert size(2, rows, 80, 16) == 80 * rows + 4 * rows + -80 * rows % 256 + -4 * rows % 256


def test_short_rows_that_two_kernels_do_sooner(native_lib):
    """Unaligned rows of the weight, and few products for a row, take a workspace."""
    size = native_lib.raw("linear_int8_workspace_size")
    for dtype in (0, 1, 2):
        assert size(dtype, 40000, 80, 128) == size(dtype, 40000, 64, 136) == size(dtype, 40000, 16, 512) == 0
        for inner, outer in ((100, 512), (3, 256), (250, 256), (64, 128), (32, 32)):
            assert size(dtype, 40000, inner, outer) > 0
