"""Ways to call the dense operators on the GPU besides the plain ones."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from muspace_amd import checkpoint_int8, layer_norm, linear

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
def test_tracing_is_refused(which, graph):
    call = calls()[which]
    x = torch.randn((3, 8), device=DEV, requires_grad=graph)
    for trace in (lambda: torch.jit.trace(call, (x,)), lambda: make_fx(call)(x.detach())):
        with pytest.raises(RuntimeError, match="HIP kernels cannot be traced"):
            trace()
    assert call(x).isfinite().all()
    with pytest.raises(RuntimeError, match="HIP kernels cannot be traced"):
        torch.jit.trace(lambda t: checkpoint_int8(t)[0], (x.detach(),))


def test_the_reference_backend_is_traced_on_the_device():
    x, w = torch.randn((3, 8), device=DEV), torch.randn((4, 8), device=DEV)
    traced = torch.jit.trace(lambda t: linear(t, w, backend="reference"), (x,))
    y = torch.randn((3, 8), device=DEV)
    torch.testing.assert_close(traced(y), linear(y, w, backend="reference"))
