"""Compile the native library in-tree for sm_100a with nvcc, and its host extension.

    python -m svox_b200.csrc.build [--force] [--verbose]

Produces ``svox_b200/csrc/libsvox_b200.so``.  Default nvcc floating-point
behaviour is kept on purpose (no --use_fast_math, IEEE division and square
root): the kernels must reproduce the reference's arithmetic.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libsvox_b200.so")
_HEADER = os.path.join("..", "..", "include", "svox_b200.h")
# the translation units, each with what it includes
UNITS = {
    "svox_b200.cu": ["common.cuh", "arith.cuh", "host.cuh", "binned.cuh", "tiles.cuh", "query.cuh",
                     "render.cuh", "render_index.cuh", "render_queue.cuh", "render_back.cuh",
                     "render_replay.cuh", "noalloc.cuh", "collective.cuh", "open_groups.h",
                     "status.h", _HEADER],
    "recurrence.cu": ["recurrence.cuh", "rays.h", "common.cuh", "arith.cuh", "status.h", _HEADER],
    "rays.cu": ["rays.cuh", "rays.h", "recurrence.cuh", "common.cuh", "arith.cuh", "status.h",
                _HEADER],
    "records.cu": ["records.cuh", "common.cuh", "arith.cuh", "status.h", _HEADER],
}


# the host side of the hot calls, a Python extension (host.cpp)
HOST_SRC = os.path.join(HERE, "host.cpp")
HOST_LIB = os.path.join(HERE, "_host.so")
HOST_DEPS = ["host.cpp", _HEADER]


def _stale(lib, deps):
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(os.path.join(HERE, d)) > t for d in deps)


def _build_host():
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-DTORCH_EXTENSION_NAME=_host", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in [*cpp_extension.include_paths(), os.path.join(cuda, "include"),
              sysconfig.get_paths()["include"]]:
        cmd += ["-isystem", d]
    cmd += ["-o", HOST_LIB, HOST_SRC]
    for d in [*cpp_extension.library_paths(), os.path.join(cuda, "lib64")]:
        cmd += ["-L" + d]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            "-lcudart"]
    subprocess.run(cmd, check=True)


def build(force=False, verbose=False):
    if force or _stale(HOST_LIB, HOST_DEPS):
        _build_host()
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    objects, running = [], []
    for unit, deps in UNITS.items():
        obj = os.path.join(HERE, unit[:-3] + ".o")
        objects.append(obj)
        if not force and not _stale(obj, [unit, *deps]):
            continue
        # (to a name of its own first: a build that is interrupted leaves no half of an object)
        part = obj + ".part"
        cmd = [nvcc, *arch, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
               *(["-Xptxas", "-v"] if verbose else []), "-c", "-o", part, os.path.join(HERE, unit)]
        running.append((subprocess.Popen(cmd), cmd, part, obj))
    for process, cmd, part, obj in running:
        if process.wait() != 0:
            raise subprocess.CalledProcessError(process.returncode, cmd)
        os.replace(part, obj)
    if running or not os.path.exists(LIB) or \
            any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objects):
        subprocess.run([nvcc, *arch, "-shared", "-o", LIB, *objects], check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
