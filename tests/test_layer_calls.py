"""Calls of the dense operators that only a part of torch sees, on the CPU: the host module
itself refuses them before anything runs."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import layer_norm, linear
from muspace_amd.runtime.layer_host import load_layer_host

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
