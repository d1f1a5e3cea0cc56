"""Builds the engine's shared library in-tree with nvcc for sm_100a, the sidecar
server (a plain C++ program over the library's C ABI) and the Python calls of
the decoder operators (an extension module against torch's headers).

``python -m cruise_b200.build`` writes ``cruise_b200/libcruise_epoch.so``,
``cruise_b200/cruise_epoch_server`` and ``cruise_b200/_decoder_bind.so``.  nvcc
cross-compiles without a GPU, so this runs on any host with CUDA 12.9; where torch
or the Python headers are missing, the extension module is left out.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
LIBRARY = PACKAGE / "libcruise_epoch.so"
SERVER = PACKAGE / "cruise_epoch_server"
SOURCES = [CSRC / "engine.cu", CSRC / "decoder_ops.cu"]
SERVER_SOURCES = [CSRC / "sidecar_server.cpp"]
BINDING = PACKAGE / "_decoder_bind.so"
BINDING_SOURCES = [CSRC / "decoder_bind.cpp"]
HEADERS = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list((PACKAGE.parent / "include").glob("*.h"))
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found: the CUDA 12.9 toolkit is required to build the engine")
    return found


def _fresh(target: Path, sources: list[Path]) -> bool:
    if not target.exists():
        return False
    built = target.stat().st_mtime
    return all(src.stat().st_mtime <= built for src in sources + HEADERS)


def up_to_date() -> bool:
    return (_fresh(LIBRARY, SOURCES) and _fresh(SERVER, SERVER_SOURCES + [LIBRARY])
            and (_fresh(BINDING, BINDING_SOURCES) or not binding_possible()))


def build_server() -> Path:
    """The sidecar server, linked against the in-tree library (found next to it)."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("a C++ compiler (g++) is required to build the sidecar server")
    tmp = SERVER.with_name(f"{SERVER.name}.tmp{os.getpid()}")
    cmd = [cxx, "-O2", "-std=c++17", "-Wall", "-o", str(tmp), *map(str, SERVER_SOURCES),
           f"-L{PACKAGE}", "-l:libcruise_epoch.so", "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, SERVER)
    return SERVER


def binding_possible() -> bool:
    """Whether this host has what the Python calls are built against; callers of
    the library in C need neither."""
    return importlib.util.find_spec("torch") is not None and Path(sysconfig.get_paths()["include"], "Python.h").exists()


def build_binding() -> Path:
    """The Python calls of the decoder operators (cruise_b200._decoder_bind)."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("a C++ compiler (g++) is required to build the decoder operators' Python calls")
    cuda = str(Path(nvcc()).resolve().parents[1] / "include")
    tmp = BINDING.with_name(f"{BINDING.name}.tmp{os.getpid()}")
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", sysconfig.get_paths()["include"], *(arg for path in [*include_paths(), cuda] for arg in ("-isystem", path)),
           "-o", str(tmp), *map(str, BINDING_SOURCES), *(f"-L{path}" for path in library_paths()),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    return BINDING


def link_flags() -> list[str]:
    """No library beyond the CUDA runtime (linked statically by nvcc); the
    driver's tensor-map encoder is found at run time through the runtime."""
    return []


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return LIBRARY
    if force or not _fresh(LIBRARY, SOURCES):
        tmp = LIBRARY.with_suffix(f".so.tmp{os.getpid()}")
        cmd = [nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-o", str(tmp), *map(str, SOURCES),
               *link_flags()]
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIBRARY)
    build_server()
    if force or not _fresh(BINDING, BINDING_SOURCES):
        if binding_possible():
            build_binding()
        else:
            print(f"{BINDING.name} not built: no torch or no Python headers here (cruise_b200.decoder_ops needs it)", file=sys.stderr)
    return LIBRARY


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
