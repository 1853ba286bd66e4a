"""Loader of the dense operators' host module, ``native/muspace_layer_host.so``.

The module holds the operators' autograd nodes (C++ against torch's API) and no
kernel; it launches through the C-ABI of ``libmuspace_msda.so``, whose addresses are
handed to it here, after that library's own checks (exports, ABI version) and the
check that the module was compiled from the same version's headers: it calls those
addresses by the headers' signatures.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from importlib.machinery import ExtensionFileLoader
from importlib.resources import files
from importlib.util import module_from_spec, spec_from_loader
from pathlib import Path

from .native import ABI_VERSION, NativeModuleUnavailable, load_native_module

MODULE_NAME = "muspace_layer_host"
_BOUND = (
    "muspace_last_error", "linear_forward", "linear_checkpoint",
    "linear_backward_workspace_size_for", "linear_backward", "layer_norm_forward",
    "layer_norm_backward_workspace_size", "layer_norm_backward", "gated_linear_forward",
    "gated_linear_backward_workspace_size", "gated_linear_backward", "quantize_int8",
    "linear_int8_workspace_size", "linear_int8_forward", "dropout_forward",
    "residual_norm_forward", "residual_norm_backward_workspace_size", "residual_norm_backward",
)


def module_path() -> Path:
    return Path(files("muspace_amd").joinpath(f"native/{MODULE_NAME}.so"))


@lru_cache(maxsize=1)
def load_layer_host():
    library = load_native_module()
    path = module_path()
    if not path.is_file():
        raise NativeModuleUnavailable(
            f"muSPACE host module is missing from this installation ({path}); "
            "build it with `python -m muspace_amd.build`."
        )
    loader = ExtensionFileLoader(MODULE_NAME, str(path))
    try:
        module = module_from_spec(spec_from_loader(MODULE_NAME, loader))
        loader.exec_module(module)
    except ImportError as exc:
        raise NativeModuleUnavailable(f"unable to load muSPACE host module {path}: {exc}") from exc
    version = getattr(module, "abi_version", None)
    if version != ABI_VERSION:
        raise NativeModuleUnavailable(
            f"muSPACE host module {path} has ABI version {version}, expected {ABI_VERSION}; "
            "rebuild it with `python -m muspace_amd.build`"
        )
    module.bind({name: ctypes.cast(library.raw(name), ctypes.c_void_p).value for name in _BOUND})
    return module


def layer_host_error() -> str | None:
    try:
        load_layer_host()
    except NativeModuleUnavailable as exc:
        return str(exc)
    return None
