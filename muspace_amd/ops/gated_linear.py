"""The first half of a gated feed-forward block: both projections, the activation and the
product in one kernel.

    a, u = input @ weight.T + bias, in halves;  out = activation(a) * u

``weight`` holds the gate's rows, then the others'. The products run on the matrix cores
with float32 sums, a and u of a result in one wavefront's registers, and neither is
written: the result is rounded once. The backward keeps the input alone and multiplies
again for a and u, a third of the products of a step more: that saves two tensors of the
block's width in memory between the passes, and the rounding that 16 bits of them would
give the gradients. It does not save time where rows are long: kept, they would be written and
read sooner. da and du are rounded to the tensors' type once, before they are multiplied with the
weight and the input.

The second half of the block is ``linear``, with its residual. No reference counterpart:
the reference leaves these products to torch.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .layer_common import DTYPES as _DTYPES
from .layer_common import in_the_tensors_type, native_for, report_native, report_other

OPERATOR_NAME = "gated_linear"
GATES = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
_FUNCTIONS = {None: lambda a: a, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
              "sigmoid": torch.sigmoid}


@in_the_tensors_type
def gated_linear_pytorch(input, weight, bias=None, *, activation="silu"):
    """``gated_linear`` in PyTorch operations, on any device."""
    a, u = F.linear(input, weight, bias).chunk(2, dim=-1)
    return _FUNCTIONS[activation](a) * u


def _validate(input, weight, bias, activation) -> None:
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if activation not in GATES:
        raise ValueError("activation must be None, 'relu', 'gelu', 'silu' or 'sigmoid', "
                         f"got {activation!r}")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if weight.dim() != 2 or weight.shape[1] != input.shape[-1] or weight.shape[0] % 2:
        raise ValueError(f"weight must be [2 * hidden_features, {input.shape[-1]}], "
                         f"got {list(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {list(bias.shape)}")
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor is not None and tensor.dtype != input.dtype:
            raise TypeError(f"{name} must be {input.dtype} like the input, got {tensor.dtype}")


def gated_linear(
    input: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = "silu",
    backend: str = "auto",
) -> torch.Tensor:
    """``activation(a) * u`` in ``input.dtype``, ``a`` and ``u`` the halves of
    ``input @ weight.T + bias``.

    ``input`` [..., in_features], ``weight`` [2 * hidden_features, in_features], the
    gate's rows first, ``bias`` [2 * hidden_features]; all of one type, float32, float16
    or bfloat16, any strides. ``activation`` of the gate: None, ``"relu"``, ``"gelu"`` (by the error
    function), ``"silu"`` or ``"sigmoid"``. Returns [..., hidden_features].

    ``backend``: ``"auto"`` (HIP kernels on ROCm tensors, the PyTorch path elsewhere),
    ``"hip"`` (native kernels or an error) or ``"reference"``. A native failure is raised,
    not hidden behind the PyTorch path. Gradients can be taken once (no gradients of
    gradients) on the HIP path.
    """
    host = native_for(input, backend)
    if host is not None and activation in GATES:
        output = host.gated_linear(input, weight, bias, GATES[activation])
        if output is not None:
            report_native(OPERATOR_NAME, input, backend)
            return output
    # not the HIP kernels' call, or tensors that do not belong together: say which
    _validate(input, weight, bias, activation)
    report_other(OPERATOR_NAME, input, backend)
    return gated_linear_pytorch(input, weight, bias, activation=activation)


__all__ = ["gated_linear", "gated_linear_pytorch"]
