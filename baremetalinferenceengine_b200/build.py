"""Compiles the sm_100a layer-op kernels into the in-tree shared library, and the Python
module over it.

    python -m baremetalinferenceengine_b200.build [--force]

produces ``baremetalinferenceengine_b200/libbm_layer_ops.so`` from ``csrc/*.cu``
with nvcc (``-gencode arch=compute_100a,code=sm_100a``), static cudart, C++17.
Objects go to ``_build/`` at the repository root. A source newer than the
library (or a changed header) triggers a rebuild. ``_serving_ops.so`` beside it is the
CPython module of ``csrc/binding/`` (g++ against torch's headers), linked to the library;
it is left out, with a note, where torch or Python's headers are not installed.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_ROOT, "include")
BUILD_DIR = os.path.join(REPO_ROOT, "_build", "bm_layer_ops")
LIB_NAME = "libbm_layer_ops.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
BINDING_SRC = os.path.join(CSRC, "binding", "serving_ops.cpp")
BINDING_PATH = os.path.join(PKG_DIR, "_serving_ops.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC,-O3",
    "--expt-relaxed-constexpr",
    "-I" + INCLUDE,
    "-I" + CSRC,
]


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build the layer-op kernels")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers() -> list[str]:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith((".h", ".cuh"))]
    return hs


def _stale(target: str, deps: list[str]) -> bool:
    if not all(os.path.exists(p) for p in [target] + deps):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError("command failed:\n  " + " ".join(cmd) + "\n" + proc.stdout)


def _binding_lacks() -> str | None:
    """What the CPython module needs and this machine has not; None where it has all."""
    if importlib.util.find_spec("torch") is None:
        return "torch is not installed"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers are not installed"
    return None


def _binding_for() -> str:
    """The torch and the Python that a module built now is for (torch itself stays unloaded)."""
    at = os.path.dirname(importlib.util.find_spec("torch").origin)
    with open(os.path.join(at, "version.py")) as f:
        return f"{at}\n{sys.implementation.cache_tag}\n{f.read()}"


def _build_binding(force: bool) -> None:
    """_serving_ops.so: g++ against torch's headers and libraries, and libbm_layer_ops.so
    (found beside it at run time). Users of the C ABI do without: where torch or Python's
    headers are missing this says so and builds nothing."""
    made_for = os.path.join(BUILD_DIR, "_serving_ops.made_for")
    lacks = _binding_lacks()
    now = "" if lacks else _binding_for()
    if not (force or _stale(BINDING_PATH, [BINDING_SRC, os.path.join(INCLUDE, "bm_layer_ops.h"), made_for])):
        with open(made_for) as f:
            if lacks or f.read() == now:
                return
    if lacks:
        print(f"{os.path.basename(BINDING_PATH)} not built: {lacks} (only the Python calls of ops.rotary, qk_norm_rotary, sample and "
              "the paged caches' need it)", file=sys.stderr)
        return
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"], INCLUDE]
    tmp = BINDING_PATH + ".tmp"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
         + [f"-I{i}" for i in includes] + [BINDING_SRC, "-o", tmp, LIB_PATH, f"-L{os.path.join(root, 'lib')}",
                                           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
                                           "-Wl,-rpath,$ORIGIN"])
    with open(made_for, "w") as f:
        f.write(now)
    os.replace(tmp, BINDING_PATH)
    os.utime(BINDING_PATH)  # not older than made_for


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds (if needed) and returns the path of libbm_layer_ops.so."""
    nvcc = nvcc_path()
    os.makedirs(BUILD_DIR, exist_ok=True)
    headers = _headers()
    objs = []
    jobs = []
    for src in sources():
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            jobs.append([nvcc] + NVCC_FLAGS + ["-c", src, "-o", obj])
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
            for f in [ex.submit(_run, j) for j in jobs]:
                f.result()
            if verbose:
                for j in jobs:
                    print(" ".join(j))
    if force or jobs or _stale(LIB_PATH, objs):
        tmp = LIB_PATH + ".tmp"
        _run([nvcc] + ARCH_FLAGS + ["-shared", "-Xlinker", f"-soname={LIB_NAME}", "-o", tmp] + objs + ["-lcudart_static", "-lrt", "-ldl", "-lpthread"])
        os.replace(tmp, LIB_PATH)
    _build_binding(force)
    return LIB_PATH


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
