"""What the layer's dense operators share: backend choice, reports and checks."""

from __future__ import annotations

from functools import lru_cache

import torch

from ..runtime.kernel_dispatch import (
    NATIVE_ALIASES,
    NATIVE_BACKEND,
    DispatchReport,
    explain_dispatch,
    is_rocm_tensor,
    record_dispatch_report,
)
from ..runtime.native import NativeModuleUnavailable, load_native_module, native_error

DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def native_library():
    """The loaded library (its bound methods, without a lookup by name per call), or None."""
    try:
        return load_native_module()
    except NativeModuleUnavailable:
        return None


def require_native():
    library = native_library()
    if library is None:
        raise RuntimeError(f"muSPACE HIP native library is unavailable: {native_error()}")
    return library


@lru_cache(maxsize=64)
def _native_report(operator: str, backend: str, device: str) -> DispatchReport:
    # reports of one operator's native calls are equal and immutable: one is enough
    reason = ("forced HIP backend" if backend in NATIVE_ALIASES
              else "ROCm tensor selects native HIP backend")
    return DispatchReport(operator, backend, NATIVE_BACKEND, device, reason, True)


def choose_native(operator: str, input: torch.Tensor, backend: str):
    """The library if the call runs on the HIP kernels, None for the PyTorch path; the
    choice is reported. Raises where neither may run."""
    library = native_library()
    if (library is not None and (backend == "auto" or backend in NATIVE_ALIASES)
            and is_rocm_tensor(input)):
        record_dispatch_report(_native_report(operator, backend, input.device.type))
        return library
    decision = explain_dispatch(input, backend=backend, native_available=library is not None)
    record_dispatch_report(DispatchReport(operator, backend, decision.backend, decision.device,
                                          decision.reason, library is not None))
    if decision.backend == "error":
        detail = native_error() if library is None and is_rocm_tensor(input) else None
        raise RuntimeError(f"{decision.reason}: {detail}" if detail else decision.reason)
    return None


def check_device(input: torch.Tensor, *named) -> None:
    """Every (tensor, name) on the input's device; None skipped."""
    device = input.device
    for tensor, name in named:
        if tensor is not None and tensor.device != device:
            raise RuntimeError(f"{name} must be a ROCm device tensor on {device} like the input, "
                               f"got device {tensor.device}")
