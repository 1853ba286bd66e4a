"""Layer norm over the last dimension, forward and backward.

The norm between the sub-layers of an encoder or decoder block: each value is
read once forward (and x and the gradient once backward), statistics in
float32, every result rounded once. The backward's weight and bias gradients
are summed over the rows in a fixed order, without atomics. For the backward the
input and two float32 numbers per row are kept.

No reference counterpart: the reference leaves norms to torch.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .layer_common import DTYPES as _DTYPES
from .layer_common import in_the_tensors_type, native_for, report_native, report_other

OPERATOR_NAME = "layer_norm"


@in_the_tensors_type
def layer_norm_pytorch(input, weight=None, bias=None, *, eps=1e-5):
    """``layer_norm`` in PyTorch operations, on any device."""
    if weight is None or weight.dtype == input.dtype:
        if bias is None or bias.dtype == input.dtype:
            return F.layer_norm(input, input.shape[-1:], weight, bias, eps)
    # float32 weights next to a 16-bit input: in float32, rounded once
    out = F.layer_norm(input.float(), input.shape[-1:],
                       None if weight is None else weight.float(),
                       None if bias is None else bias.float(), eps)
    return out.to(input.dtype)


def _validate(input, weight, bias, eps) -> None:
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor is None:
            continue
        if tensor.shape != input.shape[-1:]:
            raise ValueError(f"{name} must be [{input.shape[-1]}], got {list(tensor.shape)}")
        if tensor.dtype not in (torch.float32, input.dtype):
            raise TypeError(f"{name} must be float32 or {input.dtype}, got {tensor.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")


def layer_norm(
    input: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
    backend: str = "auto",
) -> torch.Tensor:
    """``(input - mean) / sqrt(var + eps) * weight + bias`` over the last dimension,
    in ``input.dtype`` (float32, float16 or bfloat16, any strides).

    ``weight`` and ``bias`` [cols], each optional, float32 or of the input's type;
    their gradients have their type. ``backend``: ``"auto"`` (HIP kernels on ROCm
    tensors, the PyTorch path elsewhere), ``"hip"`` (native kernels or an error) or
    ``"reference"``. A native failure is raised, not hidden behind the PyTorch path.
    Gradients can be taken once (no gradients of gradients) on the HIP path.
    """
    host = native_for(input, backend)
    if host is not None:
        output = host.layer_norm(input, weight, bias, eps)
        if output is not None:
            report_native(OPERATOR_NAME, input, backend)
            return output
    # not the HIP kernels' call, or tensors that do not belong together: say which
    _validate(input, weight, bias, eps)
    report_other(OPERATOR_NAME, input, backend)
    return layer_norm_pytorch(input, weight, bias, eps=eps)


__all__ = ["layer_norm", "layer_norm_pytorch"]
