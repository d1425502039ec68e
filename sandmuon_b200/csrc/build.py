"""Builds libsandmuon_b200.so for sm_100a with nvcc, and the torch extension of
the activation operators with g++, in-tree.

Usage:  python -m sandmuon_b200.csrc.build   (or sandmuon_b200.csrc.build.build())

The shared objects land in the package (libsandmuon_b200.so, and
_activations.<python>-torch-<version>-abi<n>.so) so they travel with the source
tree; nothing is installed into site-packages.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

from .._lib import binding_path

CSRC = Path(__file__).resolve().parent
PACKAGE = CSRC.parent
ROOT = PACKAGE.parent
LIB_NAME = "libsandmuon_b200.so"
LIB_PATH = PACKAGE / LIB_NAME
SOURCES = [CSRC / "libsandmuon_b200.cu"]
DEPENDS = SOURCES + [CSRC / "sm_common.cuh", CSRC / "sm_gemm.cuh", CSRC / "sm_kernels.cuh",
                     CSRC / "sm_activation.cuh", CSRC / "sm_wgrad.cuh", CSRC / "sm_activation_host.cuh",
                     ROOT / "include" / "sandmuon_b200.h"]

BINDING_SOURCE = CSRC / "activations_binding.cpp"
BINDING_DEPENDS = [BINDING_SOURCE, ROOT / "include" / "sandmuon_b200.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-Xptxas", "-warn-spills",
]


def nvcc_path() -> str:
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found: the sandmuon_b200 CUDA library cannot be built")


def up_to_date(target: Path = LIB_PATH, depends: list[Path] = DEPENDS) -> bool:
    if not target.exists():
        return False
    built = target.stat().st_mtime
    return all(dep.stat().st_mtime <= built for dep in depends)


def binding_command(out: Path) -> list[str]:
    """g++ command of the torch extension."""
    import torch
    from torch.utils.cpp_extension import include_paths
    # not $CXX: a toolchain that links its own libstdc++ statically gives an
    # extension whose exceptions and streams do not mix with torch's
    compiler = shutil.which("g++")
    if compiler is None:
        raise RuntimeError("g++ not found: the sandmuon_b200 torch extension cannot be built")
    cuda = Path(nvcc_path()).resolve().parents[1]
    lib = Path(torch.__file__).resolve().parent / "lib"
    includes = [*include_paths(), str(cuda / "include"), sysconfig.get_paths()["include"], str(ROOT / "include")]
    return [compiler, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            "-DTORCH_EXTENSION_NAME=_activations", "-DTORCH_API_INCLUDE_EXTENSION_H",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-I{path}" for path in includes), "-o", str(out), str(BINDING_SOURCE), f"-L{lib}",
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the library and the extension, each unless it is newer than
    every file it is made from; returns the library's path."""
    # every command is there before the first compiler starts
    jobs = []
    for target, depends, command in (
            (LIB_PATH, DEPENDS,
             lambda out: [nvcc_path(), *NVCC_FLAGS, "-I", str(ROOT / "include"), "-o", str(out), *map(str, SOURCES)]),
            (binding_path(), BINDING_DEPENDS, binding_command)):
        if force or not up_to_date(target, depends):
            tmp = target.with_suffix(".so.tmp")
            jobs.append((target, tmp, command(tmp)))
    processes = []
    try:
        for _, _, cmd in jobs:
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            processes.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
        outputs = [process.communicate()[0] for process in processes]
    finally:
        for process in processes:
            if process.poll() is None:
                process.kill()
                process.wait()
    failed = []
    for (target, tmp, _), process, output in zip(jobs, processes, outputs):
        if process.returncode != 0:
            failed.append(f"building {target.name} failed ({process.returncode}):\n{output}")
            continue
        if verbose and output:
            print(output, file=sys.stderr)
        os.replace(tmp, target)
    if failed:
        raise RuntimeError("\n".join(failed))
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
