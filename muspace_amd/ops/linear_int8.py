"""The linear layer of a deployed model in 8-bit integers.

    out = activation(input @ weight.T + bias) + residual

with each row of the input (a token) and each row of the weight (an output channel) as
8-bit codes under a float32 scale: sums of code products are exact in int32 on the matrix
cores, at twice the rate of 16-bit values, and the weight is a quarter of its float32
size. The weight is quantised once (``quantize_int8``), the input's rows in every call.

No gradients: training keeps ``linear``. No reference counterpart: the reference leaves
these products to torch.
"""

from __future__ import annotations

import torch

from .layer_common import DTYPES as _DTYPES
from .layer_common import (
    in_the_tensors_type,
    native_for,
    report_native,
    report_other,
    require_native,
    runs_native,
)
from .linear import ACTIVATIONS, _activate

OPERATOR_NAME = "linear_int8"
MAX_IN_FEATURES = 1 << 17  # sums are int32 numbers


@in_the_tensors_type
def quantize_int8_pytorch(input: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_int8`` in PyTorch operations, on any device."""
    x = input.detach().float()
    top = x.abs().amax(-1) if x.shape[-1] else x.new_zeros(x.shape[:-1])
    finite = top.isfinite()
    # (by a tensor: on a GPU torch multiplies with a number's reciprocal, which rounds twice)
    scales = torch.where(finite, (top / torch.full_like(top, 127.0)).clamp_min(2.0**-126), torch.nan)
    quotients = x / torch.where(finite, scales, 1.0).unsqueeze(-1)
    codes = torch.where(finite.unsqueeze(-1), torch.round(quotients), 1.0)
    return codes.to(torch.int8), scales


def quantize_int8(input: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``input`` [..., cols] (float32, float16 or bfloat16) by rows in 8 bits: ``(codes int8 [...,
    cols], scales float32 [...])``.

    A row's scale is its largest magnitude over 127 (at least 2^-126), its codes the
    nearest integers to value / scale, ties to even: ``codes * scales[..., None]`` is within half
    a scale of the input. A row with an infinity or NaN has scale NaN.
    """
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if runs_native(input):
        return require_native().quantize(input.detach())
    return quantize_int8_pytorch(input)


@in_the_tensors_type
def linear_int8_pytorch(input, weight, weight_scale, bias=None, *, activation=None, residual=None):
    """``linear_int8`` in PyTorch operations, on any device."""
    codes, scales = quantize_int8_pytorch(input)
    sums = codes.double() @ weight.double().t()  # integers, exact
    z = sums.float() * scales.unsqueeze(-1) * weight_scale
    if bias is not None:
        z = z + bias.float()
    out = _activate(z, activation)
    return (out if residual is None else out + residual.float()).to(input.dtype)


def _validate(input, weight, weight_scale, bias, activation, residual) -> None:
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'relu' or 'gelu', got {activation!r}")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if weight.dtype != torch.int8:
        raise TypeError(f"weight must be int8 codes, got {weight.dtype}")
    if weight.dim() != 2 or weight.shape[1] != input.shape[-1]:
        raise ValueError(f"weight must be [out_features, {input.shape[-1]}], "
                         f"got {list(weight.shape)}")
    if weight.shape[1] > MAX_IN_FEATURES:
        raise ValueError(f"in_features must be at most {MAX_IN_FEATURES}, got {weight.shape[1]}")
    if weight_scale.shape != weight.shape[:1]:
        raise ValueError(f"weight_scale must be [{weight.shape[0]}], got {list(weight_scale.shape)}")
    if weight_scale.dtype != torch.float32:
        raise TypeError(f"weight_scale must be float32, got {weight_scale.dtype}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {list(bias.shape)}")
    if residual is not None and residual.shape != (*input.shape[:-1], weight.shape[0]):
        raise ValueError(f"residual must have the output's shape "
                         f"{[*input.shape[:-1], weight.shape[0]]}, got {list(residual.shape)}")
    for name, tensor in (("bias", bias), ("residual", residual)):
        if tensor is not None and tensor.dtype != input.dtype:
            raise TypeError(f"{name} must be {input.dtype} like the input, got {tensor.dtype}")
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (input, weight_scale, bias, residual)):
        raise RuntimeError("linear_int8 has no gradients: call it under torch.no_grad() or on "
                           "tensors that require none")


def linear_int8(
    input: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    backend: str = "auto",
) -> torch.Tensor:
    """``activation(input @ weight.T + bias) + residual`` in ``input.dtype``, the products in
    8-bit integers.

    ``input`` [..., in_features] (float32, float16 or bfloat16, any strides) is quantised by
    rows in the call; ``weight`` int8 [out_features, in_features] and ``weight_scale``
    float32 [out_features] are ``quantize_int8`` of the layer's weight. ``bias`` and
    ``residual`` [..., out_features] are of the input's type. ``activation``: None, ``"relu"``
    or ``"gelu"`` (by the error function). in_features at most 2^17.

    ``backend``: ``"auto"`` (HIP kernels on ROCm tensors, the PyTorch path elsewhere),
    ``"hip"`` (native kernels or an error) or ``"reference"``. There are no gradients: a
    call on tensors that require them raises, but under ``torch.no_grad()``.
    """
    host = native_for(input, backend)
    if host is not None and activation in ACTIVATIONS and input.shape[-1:] <= (MAX_IN_FEATURES,):
        output = host.linear_int8(input, weight, weight_scale, bias, residual,
                                  ACTIVATIONS[activation])
        if output is not None:
            report_native(OPERATOR_NAME, input, backend)
            return output
    # not the HIP kernels' call, or tensors that do not belong together: say which
    _validate(input, weight, weight_scale, bias, activation, residual)
    report_other(OPERATOR_NAME, input, backend)
    return linear_int8_pytorch(input, weight, weight_scale, bias, activation=activation,
                               residual=residual)


__all__ = ["linear_int8", "linear_int8_pytorch", "quantize_int8", "quantize_int8_pytorch"]
