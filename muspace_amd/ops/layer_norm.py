"""Layer norm over the last dimension, forward and backward.

The norm between the sub-layers of an encoder or decoder block: each value is
read once forward (and x and the gradient once backward), statistics in
float32, every result rounded once. The backward's weight and bias gradients
are summed over the rows in a fixed order, without atomics. For the backward the
input and two float32 numbers per row are kept.

No reference counterpart: the reference leaves norms to torch.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .layer_common import DTYPES as _DTYPES
from .layer_common import check_device, choose_native, require_native

OPERATOR_NAME = "layer_norm"


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


class _NativeLayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, weight_dtype, eps):
        ext = require_native()
        rows = math.prod(input.shape[:-1])
        output = torch.empty_like(input)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=input.device)
        ext.layer_norm_forward_launch(input, weight, bias, weight_dtype, output, stats, rows, eps)
        # all that the backward needs to know, looked up here: its thread runs Python slowly
        ctx.launch = ext.layer_norm_backward_launch
        ctx.plan = ext.layer_norm_plan(input.dtype, weight_dtype, rows, input.shape[-1])
        ctx.weight_dtype = weight_dtype
        ctx.save_for_backward(input, weight, stats)
        return output

    @staticmethod
    def backward(ctx, grad_output):
        if torch.is_grad_enabled():  # create_graph: refuses a second differentiation
            return _layer_norm_backward_once(ctx, grad_output)
        return _layer_norm_backward(ctx, grad_output)


def _layer_norm_backward(ctx, grad_output):
    input, weight, stats = ctx.saved_tensors
    need_input, need_weight, need_bias = ctx.needs_input_grad[:3]
    grad_input = torch.empty_like(input) if need_input else None
    cols, dtype = input.shape[-1:], ctx.weight_dtype
    grad_weight = stats.new_empty(cols, dtype=dtype) if need_weight else None
    grad_bias = stats.new_empty(cols, dtype=dtype) if need_bias else None
    ctx.launch(grad_output.contiguous(), input, weight, stats, grad_input, grad_weight, grad_bias,
               ctx.plan)
    return grad_input, grad_weight, grad_bias, None, None


_layer_norm_backward_once = once_differentiable(_layer_norm_backward)


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
    _validate(input, weight, bias, eps)
    ext = choose_native(OPERATOR_NAME, input, backend)
    if ext is None:
        return layer_norm_pytorch(input, weight, bias, eps=eps)
    check_device(input, (weight, "weight"), (bias, "bias"))
    input = input.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    weight_dtype = (weight if weight is not None else bias if bias is not None else input).dtype
    if torch.is_grad_enabled() and (
            input.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _NativeLayerNormFunction.apply(input, weight, bias, weight_dtype, eps)
    output = torch.empty_like(input)
    ext.layer_norm_forward_launch(input, weight, bias, weight_dtype, output, None,
                                  math.prod(input.shape[:-1]), eps)
    return output


__all__ = ["layer_norm", "layer_norm_pytorch"]
