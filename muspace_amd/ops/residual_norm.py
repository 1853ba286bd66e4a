"""The end of a block and the start of the next: its sum with the residual stream and
the norm after it, fused with what may stand between.

    y      = post_norm(block)                        (or the block's output itself)
    stream = residual_scale * residual + gate * dropout(y)
    normed = norm(stream)

Layers that norm after their blocks go on with ``normed``, layers that norm before
with both: ``normed`` into the next block, ``stream`` past it. A gate per channel and a
norm on the block's own output are those of layers that norm on both sides or scale
their branches. Every tensor is read and written once in either direction. ``normed``
is the norm of the sum before it is rounded into ``stream``: in 16-bit types the backward
keeps the block's output and the residual and sums them again; in float32 it keeps the
stream (and the block's output for a post norm or the gate's gradient). The dropout's
mask is computed, not kept (see ``dropout``).

No reference counterpart: the reference leaves these steps to torch.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .dropout import dropped, seed_arguments, validate_seed
from .layer_common import DTYPES as _DTYPES
from .layer_common import in_the_tensors_type, native_for, report_native, report_other

OPERATOR_NAME = "residual_norm"
NORMS = {"layer": 0, "rms": 1}
POST_NORMS = {None: -1, **NORMS}


def _norm(x, kind, weight, bias, eps):
    """A norm over the last dimension, in x's type (float32)."""
    weight = None if weight is None else weight.to(x.dtype)
    bias = None if bias is None else bias.to(x.dtype)
    if kind == "layer":
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)
    out = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    out = out if weight is None else out * weight
    return out if bias is None else out + bias


@in_the_tensors_type
def residual_norm_pytorch(block, residual, weight=None, bias=None, *, norm="layer", eps=1e-5,
                          post_norm=None, post_weight=None, post_bias=None, gate=None,
                          residual_scale=1.0, dropout_p=0.0, seed=None, offset=0,
                          return_stream=True):
    """``residual_norm`` in PyTorch operations, on any device."""
    y = block.float()
    if post_norm is not None:
        y = _norm(y, post_norm, post_weight, post_bias, eps)
    y = dropped(y, dropout_p, seed, offset)
    if gate is not None:
        y = gate.float() * y
    stream = residual_scale * residual.float() + y
    normed = _norm(stream, norm, weight, bias, eps).to(block.dtype)
    return (normed, stream.to(block.dtype)) if return_stream else normed


def _validate(block, residual, vectors, norm, eps, post_norm, residual_scale, seed) -> None:
    if block.dtype not in _DTYPES:
        raise TypeError("block must be float16, bfloat16 or float32")
    if block.dim() == 0:
        raise ValueError("block must have at least one dimension")
    if residual.shape != block.shape:
        raise ValueError(f"residual must have the block's shape {list(block.shape)}, "
                         f"got {list(residual.shape)}")
    if residual.dtype != block.dtype:
        raise TypeError(f"residual must be {block.dtype} like the block, got {residual.dtype}")
    if norm not in NORMS:
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    if post_norm not in POST_NORMS:
        raise ValueError(f"post_norm must be None, 'layer' or 'rms', got {post_norm!r}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if not abs(residual_scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"residual_scale must be a finite float32 number, got {residual_scale}")
    validate_seed(seed, block)
    given = {name: tensor for name, tensor in vectors.items() if tensor is not None}
    for name, tensor in given.items():
        if name.startswith("post") and post_norm is None:
            raise ValueError(f"{name} is given without a post_norm")
        if tensor.shape != block.shape[-1:]:
            raise ValueError(f"{name} must be [{block.shape[-1]}], got {list(tensor.shape)}")
        if tensor.dtype not in (torch.float32, block.dtype):
            raise TypeError(f"{name} must be float32 or {block.dtype}, got {tensor.dtype}")
    if len({tensor.dtype for tensor in given.values()}) > 1:
        raise TypeError(f"{', '.join(given)} must be of one type, got "
                        + ", ".join(str(tensor.dtype) for tensor in given.values()))


def residual_norm(
    block: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    norm: str = "layer",
    eps: float = 1e-5,
    post_norm: str | None = None,
    post_weight: torch.Tensor | None = None,
    post_bias: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    dropout_p: float = 0.0,
    seed: int | torch.Tensor | None = None,
    offset: int = 0,
    return_stream: bool = True,
    backend: str = "auto",
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``(normed, stream)``, or ``normed`` alone without ``return_stream``:
    ``stream = residual_scale * residual + gate * dropout(post_norm(block))`` and
    ``normed = norm(stream)`` over the last dimension, both in ``block.dtype`` (float32,
    float16 or bfloat16, any strides).

    ``norm``: ``"layer"`` or ``"rms"`` (``x / sqrt(mean(x^2) + eps)``), with ``weight``
    and ``bias``; ``post_norm``: None or the same, with ``post_weight`` and
    ``post_bias`` and the same ``eps``. The vectors [cols] and ``gate`` [cols] are optional,
    all float32 or all of the block's type, as are their gradients. ``dropout_p``, ``seed``
    and ``offset`` as in ``dropout``.

    ``backend``: ``"auto"`` (HIP kernels on ROCm tensors, the PyTorch path elsewhere),
    ``"hip"`` (native kernels or an error) or ``"reference"``. A native failure is raised,
    not hidden behind the PyTorch path. Gradients can be taken once (no gradients of
    gradients) on the HIP path.
    """
    tensor, number, offset = seed_arguments(seed, offset, dropout_p)
    host = native_for(block, backend)
    if host is not None and norm in NORMS and post_norm in POST_NORMS:
        outputs = host.residual_norm(block, residual, weight, bias, gate, post_weight, post_bias,
                                     NORMS[norm], POST_NORMS[post_norm], eps, residual_scale,
                                     dropout_p, tensor, number, offset, return_stream)
        if outputs is not None:
            report_native(OPERATOR_NAME, block, backend)
            return tuple(outputs) if return_stream else outputs[0]
    # not the HIP kernels' call, or tensors that do not belong together: say which
    vectors = {"weight": weight, "bias": bias, "gate": gate, "post_weight": post_weight,
               "post_bias": post_bias}
    _validate(block, residual, vectors, norm, eps, post_norm, residual_scale, seed)
    report_other(OPERATOR_NAME, block, backend)
    return residual_norm_pytorch(block, residual, weight, bias, norm=norm, eps=eps,
                                 post_norm=post_norm, post_weight=post_weight,
                                 post_bias=post_bias, gate=gate, residual_scale=residual_scale,
                                 dropout_p=dropout_p, seed=seed, offset=offset,
                                 return_stream=return_stream)


__all__ = ["residual_norm", "residual_norm_pytorch"]
