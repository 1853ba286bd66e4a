"""Calls of the dense operators that are not the plain ones, on the CPU: what the host module
refuses before anything runs, and what the PyTorch path does in its place."""

import importlib
import math
from contextlib import nullcontext

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import (
    checkpoint_int8,
    checkpoint_restore,
    get_last_dispatch_report,
    layer_norm,
    linear,
)
from muspace_amd.runtime import native
from muspace_amd.runtime.layer_host import load_layer_host

linear_module = importlib.import_module("muspace_amd.ops.linear")  # (the package has the function)

# ------------------------------------------------- tracing, forward mode ---


def host_calls():
    """(name, call of the host module on one tensor); the rest of a call's tensors."""
    host = load_layer_host()
    w, b = torch.ones(4, 8), torch.ones(8)
    return [("linear", lambda x: host.linear(x, w, None, None, 0, False)),
            ("linear", lambda x: host.linear(x, w, None, None, 2, True)),
            ("layer_norm", lambda x: host.layer_norm(x, b, b, 1e-5)),
            ("checkpoint_int8", lambda x: host.checkpoint(x)[0])]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("graph", [False, True])
def test_host_refuses_to_be_traced(which, graph):
    name, call = host_calls()[which]
    x = torch.randn(3, 8, requires_grad=graph and which < 3)
    with pytest.raises(RuntimeError, match=f"{name}: HIP kernels cannot be traced"):
        torch.jit.trace(call, (x,))
    with pytest.raises(RuntimeError, match=f"{name}: HIP kernels cannot be traced"):
        make_fx(call)(x.detach())


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("graph", [False, True])
def test_host_refuses_forward_mode(which, graph):
    name, call = host_calls()[which]
    x = torch.randn(3, 8, requires_grad=graph)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3, 8))
        with pytest.raises(RuntimeError, match=f"{name}: the HIP path has no forward-mode"):
            call(dual)
        # the same of a view that is copied first
        dual = forward_ad.make_dual(torch.randn(8, 3), torch.ones(8, 3)).t()
        with pytest.raises(RuntimeError, match=f"{name}: the HIP path has no forward-mode"):
            call(dual)


def test_the_pytorch_path_is_traced_and_has_forward_mode():
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    traced = torch.jit.trace(lambda t: layer_norm(linear(t, w, activation="relu")), (x,))
    y = torch.randn(3, 8)
    torch.testing.assert_close(traced(y), layer_norm(linear(y, w, activation="relu")))
    with forward_ad.dual_level():
        out = linear(forward_ad.make_dual(x, torch.ones(3, 8)), w)
        torch.testing.assert_close(forward_ad.unpack_dual(out).tangent,
                                   torch.ones(3, 8) @ w.t())


# ------------------------------------------------------- the PyTorch path ---


@pytest.fixture
def device_without_library(monkeypatch, tmp_path):
    """CPU tensors count as ROCm tensors, and the host module is missing."""
    from muspace_amd.ops import layer_common
    from muspace_amd.runtime import kernel_dispatch, layer_host

    monkeypatch.setattr(layer_host, "module_path", lambda: tmp_path / "missing.so")
    monkeypatch.setattr(layer_common, "is_rocm_tensor", lambda t: True)
    monkeypatch.setattr(kernel_dispatch, "is_rocm_tensor", lambda t: True)
    if hasattr(linear_module, "is_rocm_tensor"):
        monkeypatch.setattr(linear_module, "is_rocm_tensor", lambda t: True)
    layer_host.load_layer_host.cache_clear()
    yield
    layer_host.load_layer_host.cache_clear()


def checkpointed_step(**kwargs):
    gen = torch.Generator().manual_seed(4)
    x, w = torch.randn((6, 40), generator=gen), torch.randn((5, 40), generator=gen)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = linear(xs, ws, checkpoint="int8", **kwargs)
    return [out.detach(), *torch.autograd.grad(out.square().sum(), [xs, ws]), *checkpoint_int8(x)]


def test_the_fallback_has_checkpoints(device_without_library, monkeypatch):
    """Where a missing library degrades to the PyTorch path, a checkpointed call does too."""
    with pytest.raises(RuntimeError, match="missing from this installation"):
        linear(torch.zeros(2, 4), torch.zeros(3, 4), checkpoint="int8")
    with pytest.raises(RuntimeError, match="missing from this installation"):
        checkpoint_int8(torch.zeros(2, 4))
    monkeypatch.setenv("MUSPACE_AUTO_FALLBACK", "1")
    got = checkpointed_step()
    assert get_last_dispatch_report().selected_backend == "reference"
    monkeypatch.undo()
    for a, e in zip(got, checkpointed_step()):
        assert torch.equal(a, e)


def test_the_reference_backend_needs_no_library(device_without_library):
    checkpointed = linear(torch.ones(2, 40, requires_grad=True), torch.ones(3, 40),
                          checkpoint="int8", backend="reference")
    assert torch.equal(checkpointed, torch.full((2, 3), 40.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_autocast_does_not_reach_the_pytorch_path(checkpoint, dtype):
    """Results and gradients are of the tensors' type, the same as without autocast."""
    gen = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen).to(dtype) for s in ((6, 40), (5, 40), (5,)))

    def step(mode):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        with mode:
            out = linear(*leaves, activation="gelu", checkpoint=checkpoint)
            norm = layer_norm(out, leaves[2], leaves[2])
            plain = layer_norm(out)
        # torch asks for backward passes outside of autocast
        return [out, norm, plain, *torch.autograd.grad(norm.sum() + out.sum(), leaves)]

    want = step(nullcontext())
    for other in (torch.bfloat16, torch.float16):
        for a, e in zip(step(torch.autocast("cpu", dtype=other)), want):
            assert a.dtype == dtype and torch.equal(a, e)


EMPTY = [((0, 40), 6), ((2, 0, 5), 6), ((0, 0), 6), ((3, 0), 6), ((0,), 6), ((3, 40), 0), ((0, 40), 0),
         ((40,), 6)]


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize(("shape", "outer"), EMPTY, ids=str)
def test_empty_calls_of_the_pytorch_path(shape, outer, checkpoint):
    x = torch.ones(shape, requires_grad=True)
    w, b = (torch.ones(s, requires_grad=True) for s in ((outer, shape[-1]), (outer,)))
    out = linear(x, w, b, activation="gelu", checkpoint=checkpoint)
    assert out.shape == (*shape[:-1], outer)
    dx, dw, db = torch.autograd.grad(out, [x, w, b], torch.ones_like(out))
    rows = math.prod(shape[:-1])
    assert dx.shape == shape and dw.shape == w.shape and db.shape == b.shape
    if 0 in shape:
        assert not dw.any() and not dx.any()
    codes, scales = checkpoint_int8(x)
    blocks = (shape[-1] + 31) // 32
    assert codes.shape == (rows, 32 * blocks) and scales.shape == (rows, blocks)
    assert torch.equal(checkpoint_restore(codes, scales, shape[-1], torch.float32),
                       x.detach().reshape(rows, shape[-1]))


def test_the_pytorch_path_takes_devices_without_autocast():
    x, w = torch.empty((3, 8), device="meta"), torch.empty((4, 8), device="meta")
    assert layer_norm(linear(x, w)).shape == (3, 4)


# --------------------------------------------------------- the host module ---


@pytest.mark.parametrize("version", [None, 5, 999])
def test_a_host_module_of_other_headers_is_refused(version, monkeypatch):
    """The module calls bare addresses by the signatures it was compiled with: one from before
    a change of a signature (without the attribute, or of another version) does not bind."""
    import types

    from muspace_amd.runtime import layer_host

    stale = types.SimpleNamespace(bind=lambda addresses: pytest.fail("bound"))
    if version is not None:
        stale.abi_version = version
    monkeypatch.setattr(layer_host, "module_from_spec", lambda spec: stale)
    monkeypatch.setattr(layer_host.ExtensionFileLoader, "exec_module", lambda self, module: None)
    layer_host.load_layer_host.cache_clear()
    try:
        with pytest.raises(native.NativeModuleUnavailable,
                           match=f"has ABI version {version}, expected {native.ABI_VERSION}; rebuild"):
            layer_host.load_layer_host()
    finally:
        monkeypatch.undo()
        layer_host.load_layer_host.cache_clear()
    assert layer_host.load_layer_host().abi_version == native.ABI_VERSION


def test_the_libraries_are_built_without_a_host_compiler(monkeypatch, tmp_path):
    """What the host module's build needs besides hipcc is not needed by the others."""
    from muspace_amd import build

    for name in ("LIBRARY", "PROBE_LIBRARY", "HOST_LIBRARY"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    monkeypatch.setattr(build, "build_command", lambda out, *sources: ["touch", str(out)])
    monkeypatch.setattr(build, "host_command", lambda out: ["false"])
    with pytest.raises(RuntimeError, match="building muspace_layer_host.so"):
        build.build()
    assert build.LIBRARY.is_file() and build.PROBE_LIBRARY.is_file()
    assert not build.HOST_LIBRARY.exists()
    monkeypatch.setattr(build, "host_command", lambda out: ["touch", str(out)])
    assert build.build() == build.LIBRARY and build.HOST_LIBRARY.is_file()


# ----------------------------------------------------------- the workspace ---


def test_the_workspace_is_that_of_the_wanted_gradients(native_lib):
    every = native_lib.raw("linear_backward_workspace_size")
    size = native_lib.raw("linear_backward_workspace_size_for")
    dims = (2, 80000, 512, 256)
    # 8 tiles of 128 x 128, for two workgroups on each of 256 CUs: 64 parts of 1250 steps, 20
    # steps each, which makes 63
    splits = 63
    weight, bias = splits * 256 * 512 * 4, splits * 256 * 4
    assert every(*dims, 0) == size(*dims, 0, 1, 1, 1) == weight + bias
    assert size(*dims, 0, 1, 0, 0) == size(*dims, 0, 0, 0, 0) == 0
    assert size(*dims, 0, 0, 1, 0) == size(*dims, 1, 1, 1, 0) == weight
    assert size(*dims, 0, 0, 0, 1) == size(*dims, 1, 1, 0, 1) == bias
    dz = 2 * 80000 * 256 * 2  # gelu's, for any of them
    assert size(*dims, 2, 1, 0, 0) == dz and size(*dims, 2, 0, 0, 1) == dz + bias
    assert size(*dims, 2, 0, 0, 0) == 0 and every(*dims, 2) == dz + weight + bias
    assert size(9, 80000, 512, 256, 0, 1, 1, 1) == 0
