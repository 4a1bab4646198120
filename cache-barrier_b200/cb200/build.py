"""Build the sm_100a kernel library ``libcb200.so`` in-tree.

``python -m cb200.build`` (with ``cache-barrier_b200`` on ``sys.path``) or
``cb200.build.build()`` compiles every ``csrc/*.cu`` with nvcc for
``compute_100a/sm_100a`` and links one shared library next to this file. The
library exports the C ABI declared in ``include/cb200.h`` and links the CUDA
runtime statically, so it loads with ``ctypes`` alone.

``csrc/torch_binding.cpp`` (the native torch layer of the decoder-layer operators)
is compiled with the host compiler against the installed torch into ``_native.so``, and
again when another torch or Python is installed. Without torch only the library is built.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(HERE)                    # cache-barrier_b200/
REPO_ROOT = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO_ROOT, "include")
OBJ_DIR = os.path.join(PKG_ROOT, "_build")
LIB_PATH = os.path.join(HERE, "libcb200.so")
NATIVE_SRC = os.path.join(CSRC, "torch_binding.cpp")
NATIVE_PATH = os.path.join(HERE, "_native.so")
NATIVE_STAMP = os.path.join(OBJ_DIR, "native.stamp")  # what _native.so was compiled against

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
                           "-Xcompiler", "-fvisibility=hidden", "-I" + INCLUDE, "-I" + CSRC]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the sm_100a kernels cannot be built")
    return cand


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs.append(os.path.join(INCLUDE, "cb200.h"))
    return hs


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _native_command():
    """(compiler command, what the result depends on besides its sources); None without torch."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return None
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("g++ not found: the native torch layer cannot be built")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + sysconfig.get_paths()["include"],
           "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I" + os.path.join(cuda, "include"), "-I" + INCLUDE, NATIVE_SRC, "-o", NATIVE_PATH,
           "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    return cmd, "\n".join([torch.__version__, sys.version, os.path.dirname(sys.executable), root])


def _read(path: str) -> str | None:
    if not os.path.exists(path):
        return None
    with open(path) as f:
        return f.read()


def build(verbose: bool = False, force: bool = False) -> str:
    """Compile (if stale) the library and, where torch is installed, the native torch layer;
    the path of ``libcb200.so``."""
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    headers = _headers()
    jobs = []
    objs = []
    for src in _sources():
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            jobs.append([nvcc] + NVCC_FLAGS + ["-c", src, "-o", obj])

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        if verbose:
            sys.stdout.write(r.stdout + r.stderr)
        return cmd

    compiled = bool(jobs)
    native = _native_command()
    if native is not None:
        if force or _stale(NATIVE_PATH, [NATIVE_SRC, os.path.join(INCLUDE, "cb200.h")]) or _read(NATIVE_STAMP) != native[1]:
            jobs.append(native[0])
        else:
            native = None
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            list(ex.map(run, jobs))
    if native is not None:
        with open(NATIVE_STAMP, "w") as f:
            f.write(native[1])
    if force or compiled or _stale(LIB_PATH, objs):
        cmd = [nvcc] + ARCH_FLAGS + ["-shared", "-o", LIB_PATH] + objs + ["-lcudart_static", "-ldl", "-lrt", "-lpthread"]
        run(cmd)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
