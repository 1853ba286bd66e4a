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

from ..runtime.kernel_dispatch import (
    NATIVE_BACKEND,
    DispatchReport,
    explain_dispatch as _explain_dispatch,
    is_rocm_tensor,
    record_dispatch_report,
)
from ..runtime.native import native_error
from .multi_scale_deformable_attn import _native_extension

OPERATOR_NAME = "layer_norm"

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


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
    def forward(ctx, input, weight, bias, eps):
        ext = _native_extension()
        if ext is None:
            raise RuntimeError("muSPACE HIP native library is unavailable")
        rows = math.prod(input.shape[:-1])
        output = torch.empty_like(input)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=input.device)
        ext.layer_norm_forward(input, weight, bias, output, stats, eps)
        ctx.weight_dtype = (weight if weight is not None else bias if bias is not None
                            else input).dtype
        ctx.save_for_backward(input, weight, stats)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        ext = _native_extension()
        if ext is None:
            raise RuntimeError("muSPACE HIP native library is unavailable")
        input, weight, stats = ctx.saved_tensors
        need_input, need_weight, need_bias = ctx.needs_input_grad[:3]
        cols = input.shape[-1]

        def column_gradient(wanted):
            if not wanted:
                return None
            return torch.empty(cols, dtype=ctx.weight_dtype, device=input.device)

        grad_input = torch.empty_like(input) if need_input else None
        grad_weight, grad_bias = column_gradient(need_weight), column_gradient(need_bias)
        ext.layer_norm_backward(grad_output.contiguous(), input, weight, stats, grad_input,
                                grad_weight, grad_bias)
        return grad_input, grad_weight, grad_bias, None


def _report(backend, selected, decision, native_available):
    record_dispatch_report(
        DispatchReport(
            operator=OPERATOR_NAME,
            requested_backend=backend,
            selected_backend=selected,
            device=decision.device,
            reason=decision.reason,
            native_available=native_available,
        )
    )


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
    ext = _native_extension()
    decision = _explain_dispatch(input, backend=backend, native_available=ext is not None)
    if decision.backend == "error":
        _report(backend, "error", decision, ext is not None)
        detail = native_error() if ext is None and is_rocm_tensor(input) else None
        raise RuntimeError(f"{decision.reason}: {detail}" if detail else decision.reason)
    if decision.backend == "reference":
        _report(backend, "reference", decision, ext is not None)
        return layer_norm_pytorch(input, weight, bias, eps=eps)
    input = input.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (input, weight, bias)):
        output = _NativeLayerNormFunction.apply(input, weight, bias, eps)
    else:
        output = torch.empty_like(input)
        ext.layer_norm_forward(input, weight, bias, output, None, eps)
    _report(backend, NATIVE_BACKEND, decision, True)
    return output


__all__ = ["layer_norm", "layer_norm_pytorch"]
