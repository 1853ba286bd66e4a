"""Build the gfx950 C-ABI library ``muspace_amd/native/libmuspace_msda.so``.

Replaces the reference's ``mcc`` + TVM-FFI AOT build
(/root/reference/native_build.py:27-65, sources listed in
/root/reference/build_utils.py:12-30) with one ``hipcc`` invocation over the
HIP sources in ``muspace_amd/csrc``. The library is built in-tree so that it
travels with the source tree; ``python -m muspace_amd.build`` rebuilds it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_DIR = PACKAGE_DIR.parent
SOURCES = (
    PACKAGE_DIR / "csrc" / "msda_capi.hip",
    PACKAGE_DIR / "csrc" / "dfa_capi.hip",
    PACKAGE_DIR / "csrc" / "linear_capi.hip",
    PACKAGE_DIR / "csrc" / "layer_norm_capi.hip",
)
DEPENDS = (
    PACKAGE_DIR / "csrc" / "capi_errors.hpp",
    PACKAGE_DIR / "csrc" / "msda_device.hpp",
    PACKAGE_DIR / "csrc" / "msda_kernels.hpp",
    PACKAGE_DIR / "csrc" / "msda_backward_tiles.hpp",
    PACKAGE_DIR / "csrc" / "msda_forward_bin.hpp",
    PACKAGE_DIR / "csrc" / "msda_forward_slab.hpp",
    PACKAGE_DIR / "csrc" / "dfa_kernels.hpp",
    PACKAGE_DIR / "csrc" / "linear_device.hpp",
    PACKAGE_DIR / "csrc" / "linear_kernels.hpp",
    PACKAGE_DIR / "csrc" / "layer_norm_kernels.hpp",
    REPO_DIR / "include" / "muspace_msda.h",
    REPO_DIR / "include" / "muspace_dfa.h",
    REPO_DIR / "include" / "muspace_layer.h",
)
LIBRARY = PACKAGE_DIR / "native" / "libmuspace_msda.so"
# memory-system probes for bench.py (--gather-probe, --atomic-probe); not
# loaded by the operators
PROBE_SOURCES = (PACKAGE_DIR / "csrc" / "probes.hip",)
PROBE_LIBRARY = PACKAGE_DIR / "native" / "libmuspace_probes.so"
# autograd nodes of the layer's dense operators: host code against torch's C++ API,
# no kernels (muspace_amd/runtime/layer_host.py loads it)
HOST_SOURCES = (PACKAGE_DIR / "csrc" / "layer_host.cpp",)
HOST_LIBRARY = PACKAGE_DIR / "native" / "muspace_layer_host.so"
OFFLOAD_ARCH = "gfx950"

# -packed-fp32-ops keeps the compiler from emitting packed fp32 VALU
# instructions (v_pk_*_f32); every kernel here is memory-bound, so nothing is
# lost.
HIPCC_FLAGS = (
    f"--offload-arch={OFFLOAD_ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-fvisibility=hidden",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wall",
)


def hipcc() -> str:
    found = shutil.which("hipcc")
    if found:
        return found
    fallback = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "bin" / "hipcc"
    if fallback.is_file():
        return str(fallback)
    raise FileNotFoundError("hipcc not found; ROCm is required to build libmuspace_msda.so")


def build_command(output: Path, sources=SOURCES) -> list[str]:
    return [hipcc(), *HIPCC_FLAGS, *(str(s) for s in sources), "-o", str(output)]


def host_command(output: Path) -> list[str]:
    """The C++ compiler's command for the host module, with torch's own headers and ABI."""
    import torch
    from torch.utils import cpp_extension

    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                f"{rocm}/include"]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return [
        os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
        "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
        *(arg for path in includes for arg in ("-isystem", path)),
        *(str(source) for source in HOST_SOURCES), "-o", str(output),
        *(f"-L{path}" for path in cpp_extension.library_paths()),
        "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip",
    ]


def _compile(library: Path, command, verbose: bool) -> Path:
    """Run ``command(output)`` into a file beside ``library``, then move it there."""
    library.parent.mkdir(parents=True, exist_ok=True)
    tmp = library.with_name(library.name + f".tmp{os.getpid()}")
    cmd = command(tmp)
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        tmp.unlink(missing_ok=True)
        raise RuntimeError(
            f"{Path(cmd[0]).name} failed ({proc.returncode}) building {library.name}:\n{proc.stderr[-4000:]}"
        )
    os.replace(tmp, library)
    return library


def build(verbose: bool = False) -> Path:
    """Compile the MSDA library, the probe library and the host module (always), each
    moved into place atomically; returns the MSDA library's path. The host module comes
    last: without a C++ compiler or torch's headers it is the only one that fails, and
    only the operators it holds are not there."""
    _compile(LIBRARY, build_command, verbose)
    _compile(PROBE_LIBRARY, lambda out: build_command(out, PROBE_SOURCES), verbose)
    _compile(HOST_LIBRARY, host_command, verbose)
    return LIBRARY


def main(argv: list[str] | None = None) -> int:
    args = sys.argv[1:] if argv is None else argv
    path = build(verbose="-v" in args or "--verbose" in args)
    print(path)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
