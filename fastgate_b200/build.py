"""In-tree build of the native parts of fastgate_b200 (sm_100a only).

  libfastgate_b200.so   CUDA kernels + C ABI (nvcc; no PyTorch dependency)
  _C.so                 pybind11/torch extension exposing the reference's operator names,
                        a thin layer over the C ABI (g++, links libfastgate_b200.so)

Both land next to this file so that they travel with the source tree.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfastgate_b200.so")
EXT = os.path.join(HERE, "_C.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]
# translation units of libfastgate_b200.so
LIB_SOURCES = ("fg_capi.cu", "fg_plan.cpp", "fg_norm.cu", "fg_linear8.cu", "fg_kv4.cu", "fg_attn4.cu")
# translation units of the pybind extension
EXT_SOURCES = ("fg_torch.cpp", "fg_torch_serving.cpp", "fg_torch_graph.cpp")


def _newer(target: str, sources: list[str]) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(s) <= t for s in sources)


def _with_includes(path: str, seen: set[str] | None = None) -> set[str]:
    """`path` and every file of this repository that it includes, directly or through others."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path in seen or not os.path.exists(path):
        return seen
    seen.add(path)
    with open(path) as f:
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', f.read(), flags=re.M):
            _with_includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: fastgate_b200 needs the CUDA 12.9 toolkit to build")
    return cand


def _object(source: str) -> str:
    return os.path.join(CSRC, os.path.splitext(source)[0] + ".o")


def _compile(sources: tuple[str, ...], command, force: bool) -> list[str]:
    """Objects of `sources`, those that are out of date compiled side by side (`command(src, obj)`)."""
    running = []
    for name in sources:
        src, obj = os.path.join(CSRC, name), _object(name)
        if not force and _newer(obj, sorted(_with_includes(src))):
            continue
        if os.path.exists(obj):
            os.remove(obj)  # an interrupted compilation leaves no stale object behind
        cmd = command(src, obj)
        running.append((cmd, subprocess.Popen(cmd, cwd=CSRC)))
    failed = [cmd for cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    return [_object(name) for name in sources]


def build_lib(force: bool = False, verbose: bool = False) -> str:
    deps = set()
    for name in LIB_SOURCES:
        deps |= _with_includes(os.path.join(CSRC, name))
    if not force and _newer(LIB, sorted(deps)):
        return LIB
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else [])
    objs = _compile(LIB_SOURCES, lambda src, obj: [nvcc_path(), *flags, "-c", "-o", obj, src], force)
    subprocess.run([nvcc_path(), *NVCC_FLAGS, "-shared", "-o", LIB, *objs], check=True, cwd=CSRC)
    return LIB


def build_ext(force: bool = False) -> str:
    """pybind11 torch extension; compiled with g++ against the installed torch headers."""
    build_lib(force=False)
    deps = {LIB}
    for name in EXT_SOURCES:
        deps |= _with_includes(os.path.join(CSRC, name))
    if not force and _newer(EXT, sorted(deps)):
        return EXT
    import torch
    from torch.utils import cpp_extension as ce

    inc = []
    for p in ce.include_paths(device_type="cuda") if "device_type" in ce.include_paths.__code__.co_varnames else ce.include_paths(cuda=True):
        inc += ["-isystem", p]
    inc += ["-isystem", sysconfig.get_paths()["include"]]
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cxx11 = int(getattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", True))
    flags = ["-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={cxx11}", "-DTORCH_EXTENSION_NAME=_C",
             "-DTORCH_API_INCLUDE_EXTENSION_H"]
    objs = _compile(EXT_SOURCES, lambda src, obj: ["g++", *flags, *inc, "-c", src, "-o", obj], force)
    cmd = [
        "g++", "-shared", *objs, "-o", EXT,
        f"-L{HERE}", "-lfastgate_b200", "-Wl,-rpath,$ORIGIN",
        f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-lc10", "-ltorch_python", "-lc10_cuda", "-ltorch_cuda",
        f"-Wl,-rpath,{torch_lib}",
    ]
    subprocess.run(cmd, check=True, cwd=CSRC)
    return EXT


def build_all(force: bool = False) -> None:
    build_lib(force)
    build_ext(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print(LIB)
    print(EXT)
