"""What the layer's dense operators share: backend choice and reports."""

from __future__ import annotations

from functools import lru_cache, wraps
from inspect import signature

import torch

from ..runtime.kernel_dispatch import (
    NATIVE_ALIASES,
    NATIVE_BACKEND,
    DispatchReport,
    explain_dispatch,
    is_rocm_tensor,
    record_dispatch_report,
)
from ..runtime.layer_host import layer_host_error, load_layer_host
from ..runtime.native import NativeModuleUnavailable

DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _native():
    try:
        return load_layer_host()
    except NativeModuleUnavailable:
        return None


def require_native():
    """The host module with the operators' autograd nodes; RuntimeError without one."""
    host = _native()
    if host is None:
        raise RuntimeError(f"muSPACE HIP native library is unavailable: {layer_host_error()}")
    return host


def runs_native(input: torch.Tensor) -> bool:
    """Whether ``backend="auto"`` takes the HIP kernels for ``input`` (or raises without
    them), not the PyTorch path."""
    if not is_rocm_tensor(input):
        return False
    return explain_dispatch(input, native_available=_native() is not None).backend != "reference"


def in_the_tensors_type(function):
    """A PyTorch path that computes in its tensors' type, as the kernels do: autocast, which
    would choose another, is off within it."""

    first = next(iter(signature(function).parameters))

    @wraps(function)
    def call(*args, **kwargs):
        device = (args[0] if args else kwargs[first]).device.type
        if not torch.amp.is_autocast_available(device) or not torch.is_autocast_enabled(device):
            return function(*args, **kwargs)
        with torch.autocast(device, enabled=False):
            return function(*args, **kwargs)

    return call


@lru_cache(maxsize=64)
def _native_report(operator: str, backend: str, device: str) -> DispatchReport:
    # reports of one operator's native calls are equal and immutable: one is enough
    reason = ("forced HIP backend" if backend in NATIVE_ALIASES
              else "ROCm tensor selects native HIP backend")
    return DispatchReport(operator, backend, NATIVE_BACKEND, device, reason, True)


def report_native(operator: str, input: torch.Tensor, backend: str) -> None:
    record_dispatch_report(_native_report(operator, backend, input.device.type))


def native_for(input: torch.Tensor, backend: str):
    """The host module if a call on ``input`` runs on the HIP kernels, else None."""
    if (backend == "auto" or backend in NATIVE_ALIASES) and is_rocm_tensor(input):
        return _native()
    return None


def report_other(operator: str, input: torch.Tensor, backend: str) -> None:
    """Reports the PyTorch path of a call that :func:`native_for` gives no module for;
    raises, with a report, where that path may not run."""
    host = _native()
    decision = explain_dispatch(input, backend=backend, native_available=host is not None)
    record_dispatch_report(DispatchReport(operator, backend, decision.backend, decision.device,
                                          decision.reason, host is not None))
    if decision.backend == "error":
        detail = layer_host_error() if host is None and is_rocm_tensor(input) else None
        raise RuntimeError(f"{decision.reason}: {detail}" if detail else decision.reason)
