"""The linear layer of an encoder or decoder block, with its epilogue fused.

Deformable-attention layers surround the attention with dense products: value,
offset, weight and output projections and a feed-forward block, each followed by
a bias, sometimes an activation, often the layer's input:

    out = activation(input @ weight.T + bias) + residual

``linear`` computes this in one kernel, on the matrix cores with float32 sums,
rounded once. Its backward recomputes nothing and keeps little: relu keeps one
bit per value (not the output), gelu its derivative in the type's size, and the input either
as it is or, with ``checkpoint="int8"``, in 8 bits: blocks of 32 values share a
power of two, and the weight's gradient is the product with exactly the values
that were kept (``checkpoint_int8``, ``checkpoint_restore``). Such a call keeps
1.03 bytes of input per value instead of 2 or 4; every other result is the
same as without. The input's gradient needs no input at all.

No reference counterpart: the reference leaves these products to torch
(/root/reference/mu_space/ops/multi_scale_deformable_attn.py:215-338 starts at the projected value).
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .layer_common import DTYPES as _DTYPES
from .layer_common import (
    in_the_tensors_type,
    native_for,
    report_native,
    report_other,
    require_native,
    runs_native,
)

OPERATOR_NAME = "linear"
BLOCK = 32  # values of a row that share a scale in an 8-bit checkpoint
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2}

# by type: the smallest scale exponent, and the one whose codes end at 63 since
# 64 * 2^e is past the type's largest number
_SCALE_RANGE = {torch.float16: (-24, 10), torch.bfloat16: (-126, 122), torch.float32: (-126, 122)}


# ------------------------------------------------------------- checkpoints ---


def _checkpoint_pytorch(input: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``checkpoint_int8`` in PyTorch operations, on any device."""
    cols = input.shape[-1]
    rows = math.prod(input.shape[:-1])
    padded = (cols + BLOCK - 1) // BLOCK * BLOCK
    low, high = _SCALE_RANGE[input.dtype]
    x = F.pad(input.reshape(rows, cols).float(), (0, padded - cols))
    x = x.view(rows, padded // BLOCK, BLOCK)
    finite = torch.isfinite(x).all(-1, keepdim=True)
    mantissa, exponent = torch.frexp(torch.where(finite, x, 0.0).abs().amax(-1, keepdim=True))
    exponent = (exponent - 7 + (mantissa > 127.0 / 128.0).int()).clamp_min(low)
    exponent = torch.where(mantissa == 0, low, exponent)  # a block of zeros
    limit = torch.where(exponent >= high, 63.0, 127.0)
    # 2^-e from its bits (a power function may be off by its last one, which would show at
    # ties): e is in [-126, 122]
    codes = (x * ((127 - exponent) << 23).view(torch.float32)).round()
    codes = torch.where(finite, torch.minimum(torch.maximum(codes, -limit), limit), 1.0)
    scales = torch.where(finite, exponent + 127, 255)
    return codes.view(rows, padded).to(torch.int8), scales.squeeze(-1).to(torch.uint8)


def checkpoint_int8(input: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``input`` [..., cols] in 8 bits: ``(codes int8 [rows, padded], scales
    uint8 [rows, padded / 32])``, cols padded to a multiple of 32.

    A block of 32 values of a row shares 2^e, the smallest power of two with
    127 * 2^e at or over the block's largest magnitude; a code is x / 2^e
    rounded to the nearest integer, ties to even; a scale byte is e + 127, or 255
    where the block holds an infinity or NaN: it reads back as NaN.
    """
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if runs_native(input):
        return require_native().checkpoint(input.detach())
    return _checkpoint_pytorch(input.detach())


def checkpoint_restore(codes: torch.Tensor, scales: torch.Tensor, cols: int,
                       dtype: torch.dtype) -> torch.Tensor:
    """The values an 8-bit checkpoint stands for, ``[rows, cols]`` in ``dtype``
    (exact: a code times its power of two is a number of the type)."""
    rows, padded = codes.shape
    exponent = scales.to(torch.int32) - 127
    # 2^e straight from its bits: e is in [-126, 122]
    factor = ((exponent + 127).clamp(1, 254) << 23).view(torch.float32)
    factor = torch.where(scales == 255, math.nan, factor)
    values = codes.view(rows, padded // BLOCK, BLOCK).float() * factor.unsqueeze(-1)
    return values.view(rows, padded)[:, :cols].to(dtype)


# ---------------------------------------------------------- PyTorch path ---


def _activate(z: torch.Tensor, activation: str | None) -> torch.Tensor:
    if activation == "relu":
        return F.relu(z)
    if activation == "gelu":
        return F.gelu(z)
    return z


class _CheckpointedInput(torch.autograd.Function):
    """``F.linear`` whose backward reads the input from its 8-bit checkpoint."""

    @staticmethod
    def forward(ctx, input, weight):
        ctx.shape, ctx.dtype = input.shape, input.dtype
        ctx.save_for_backward(weight, *_checkpoint_pytorch(input))
        return F.linear(input, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, codes, scales = ctx.saved_tensors
        kept = checkpoint_restore(codes, scales, ctx.shape[-1], ctx.dtype)
        flat = grad.reshape(kept.shape[0], grad.shape[-1])
        return grad @ weight, flat.t() @ kept


@in_the_tensors_type
def linear_pytorch(input, weight, bias=None, *, activation=None, residual=None, checkpoint=None):
    """``linear`` in PyTorch operations, on any device."""
    if checkpoint is None:
        z = F.linear(input, weight, bias)
    else:
        z = _CheckpointedInput.apply(input, weight)
        if bias is not None:
            z = z + bias
    out = _activate(z, activation)
    return out if residual is None else out + residual


# ---------------------------------------------------------------- operator ---


def _validate(input, weight, bias, activation, residual, checkpoint) -> None:
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'relu' or 'gelu', got {activation!r}")
    if checkpoint is not None and checkpoint != "int8":
        raise ValueError(f"checkpoint must be None or 'int8', got {checkpoint!r}")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    if weight.dim() != 2 or weight.shape[1] != input.shape[-1]:
        raise ValueError(f"weight must be [out_features, {input.shape[-1]}], "
                         f"got {list(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {list(bias.shape)}")
    if residual is not None and residual.shape != (*input.shape[:-1], weight.shape[0]):
        raise ValueError(f"residual must have the output's shape "
                         f"{[*input.shape[:-1], weight.shape[0]]}, got {list(residual.shape)}")
    for name, tensor in (("weight", weight), ("bias", bias), ("residual", residual)):
        if tensor is not None and tensor.dtype != input.dtype:
            raise TypeError(f"{name} must be {input.dtype} like the input, got {tensor.dtype}")


def linear(
    input: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    checkpoint: str | None = None,
    backend: str = "auto",
) -> torch.Tensor:
    """``activation(input @ weight.T + bias) + residual``, in ``input.dtype``.

    ``input`` [..., in_features], ``weight`` [out_features, in_features], ``bias``
    [out_features], ``residual`` of the output's shape [..., out_features]; all of
    one type, float32, float16 or bfloat16, any strides. ``activation``: None,
    ``"relu"`` or ``"gelu"`` (by the error function). ``checkpoint="int8"`` keeps the
    input for the weight's gradient in 8 bits (see the module's text).

    ``backend``: ``"auto"`` (HIP kernels on ROCm tensors, the PyTorch path
    elsewhere), ``"hip"`` (native kernels or an error) or ``"reference"``. A native
    failure is raised, not hidden behind the PyTorch path. Gradients can be taken
    once (no gradients of gradients) on the HIP path.
    """
    host = native_for(input, backend)
    if host is not None and activation in ACTIVATIONS and checkpoint in (None, "int8"):
        output = host.linear(input, weight, bias, residual, ACTIVATIONS[activation],
                             checkpoint is not None)
        if output is not None:
            report_native(OPERATOR_NAME, input, backend)
            return output
    # not the HIP kernels' call, or tensors that do not belong together: say which
    _validate(input, weight, bias, activation, residual, checkpoint)
    report_other(OPERATOR_NAME, input, backend)
    return linear_pytorch(input, weight, bias, activation=activation, residual=residual,
                          checkpoint=checkpoint)


__all__ = ["checkpoint_int8", "checkpoint_restore", "linear", "linear_pytorch"]
