"""Dropout from a counter-based generator, whose mask is never stored.

    out = kept * input / (1 - p) + residual

Whether element i (of the tensor in row-major order) is kept follows from ``seed``,
``offset`` and i alone: word i % 4 of Philox4x32-10 (Salmon et al., "Parallel random
numbers: as easy as 1, 2, 3", 2011) at counter (i // 4, offset) under the key ``seed``
is at or over p 2^32. The backward computes the mask again, so a call keeps nothing for
it but these numbers. Calls of one step take different offsets, steps different seeds:
the same pair draws the same mask, which is also how a recomputed block gets its own.

No reference counterpart: the reference leaves dropout to torch.
"""

from __future__ import annotations

import torch

from .layer_common import DTYPES as _DTYPES
from .layer_common import in_the_tensors_type, native_for, report_native, report_other

OPERATOR_NAME = "dropout"
_MASK32 = 0xFFFFFFFF


def seed_arguments(seed, offset, p):
    """(seed tensor or None, seed, offset) as the host module takes them; a call without
    dropout needs no seed. ValueError or TypeError for others."""
    if p == 0.0 and seed is None and offset == 0:  # a call without dropout
        return None, 0, 0
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must be in [0, 1], got {p}")
    if not isinstance(offset, int) or not 0 <= offset < 1 << 64:
        raise ValueError(f"offset must be an integer in [0, 2^64), got {offset!r}")
    if isinstance(seed, torch.Tensor):
        return seed, 0, offset
    if seed is None and p == 0.0:
        return None, 0, offset
    if not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError("seed must be an integer in [0, 2^64) or an int64 tensor of one element, "
                         f"got {seed!r}")
    return None, seed, offset


def validate_seed(seed, input) -> None:
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise TypeError("a seed tensor must hold one int64 element, got "
                            f"{list(seed.shape)} of {seed.dtype}")
        if seed.device != input.device:
            raise RuntimeError(f"seed must be on {input.device} like the input, got {seed.device}")


def kept_elements(shape, p, seed, offset, device) -> torch.Tensor:
    """The mask of a call: True where an element is kept."""
    count = torch.Size(shape).numel()
    if isinstance(seed, torch.Tensor):
        key = seed.reshape(())
    else:
        # the 64 bits as torch holds them, signed
        key = torch.tensor(seed - (1 << 64) if seed >> 63 else seed, dtype=torch.int64,
                           device=device)
    index = torch.arange((count + 3) // 4, device=device)
    c0, c1 = index & _MASK32, index >> 32
    c2, c3 = torch.full_like(index, offset & _MASK32), torch.full_like(index, offset >> 32)
    k0, k1 = key & _MASK32, (key >> 32) & _MASK32
    for _ in range(10):
        # products wrap around in 64 bits, which keeps both halves of their own 64
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & _MASK32) ^ c1 ^ k0, p1 & _MASK32,
                          ((p0 >> 32) & _MASK32) ^ c3 ^ k1, p0 & _MASK32)
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    words = torch.stack((c0, c1, c2, c3), -1).view(-1)[:count]
    return (words >= round(p * 2.0**32)).view(shape)


def dropped(values: torch.Tensor, p, seed, offset) -> torch.Tensor:
    """``values`` (float32) with the call's elements dropped and the others scaled."""
    if p == 0.0:
        return values
    kept = kept_elements(values.shape, p, seed, offset, values.device)
    scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    return torch.where(kept, values * scale, 0.0)


@in_the_tensors_type
def dropout_pytorch(input, p, *, seed=None, offset=0, residual=None):
    """``dropout`` in PyTorch operations, on any device."""
    out = dropped(input.float(), p, seed, offset)
    if residual is not None:
        out = out + residual.float()
    return out.to(input.dtype)


def _validate(input, seed, residual) -> None:
    if input.dtype not in _DTYPES:
        raise TypeError("input must be float16, bfloat16 or float32")
    validate_seed(seed, input)
    if residual is not None:
        if residual.shape != input.shape:
            raise ValueError(f"residual must have the input's shape {list(input.shape)}, "
                             f"got {list(residual.shape)}")
        if residual.dtype != input.dtype:
            raise TypeError(f"residual must be {input.dtype} like the input, got {residual.dtype}")


def dropout(
    input: torch.Tensor,
    p: float,
    *,
    seed: int | torch.Tensor | None,
    offset: int = 0,
    residual: torch.Tensor | None = None,
    backend: str = "auto",
) -> torch.Tensor:
    """``input / (1 - p)`` where an element is kept, 0 elsewhere, plus ``residual``, in
    ``input.dtype`` (float32, float16 or bfloat16, any strides).

    ``p`` in [0, 1], exact to 2^-32. ``seed``: an integer of 64 bits (may be None with
    p 0), or an int64 tensor of one element on the input's device, which the kernels read: a step
    captured into a graph draws new masks when the tensor changes between replays (not
    between a forward and its backward). ``offset``: an integer of 64 bits, of the
    call's own within a step. What is dropped is 0, whatever it was.

    ``backend``: ``"auto"`` (HIP kernels on ROCm tensors, the PyTorch path elsewhere),
    ``"hip"`` (native kernels or an error) or ``"reference"``; all draw the same
    masks. Gradients can be taken once (no gradients of gradients) on the HIP path.
    """
    tensor, number, offset = seed_arguments(seed, offset, p)
    host = native_for(input, backend)
    if host is not None:
        output = host.dropout(input, residual, p, tensor, number, offset)
        if output is not None:
            report_native(OPERATOR_NAME, input, backend)
            return output
    # not the HIP kernels' call, or tensors that do not belong together: say which
    _validate(input, seed, residual)
    report_other(OPERATOR_NAME, input, backend)
    return dropout_pytorch(input, p, seed=seed, offset=offset, residual=residual)


__all__ = ["dropout", "dropout_pytorch"]
