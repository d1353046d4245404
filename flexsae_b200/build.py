"""Builds the CUDA library in-tree: ``flexsae_b200/_lib/libflexsae_b200.so`` for sm_100a, and the Python
binding of its optimizer entry points (``csrc/host``, plain C++ against torch) beside it.

nvcc cross-compiles without a GPU, so this runs on a CPU-only machine; the shared object then
travels with the source tree.  ``python -m flexsae_b200.build`` rebuilds when a source is newer
than the library; ``--force`` always rebuilds; ``--verbose`` prints ptxas resource usage;
``--trace`` builds the tuning variant ``libflexsae_b200_trace.so`` (compiled with
``-DFLEXSAE_TRACE``: the sharded backward records a per-slot timeline, see ``slot_timeline.py``).
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libflexsae_b200.so")
TRACE_LIB_PATH = os.path.join(LIB_DIR, "libflexsae_b200_trace.so")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
]
#: sources compiled without ``--use_fast_math``: the optimizer's 8-bit states are rounded on bit patterns
#: that flush-to-zero would destroy, and its 32-bit update uses IEEE division and square root
IEEE_SOURCES = ("flexsae_optim.cu", "flexsae_optim_rows.cu")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale(lib_path: str = LIB_PATH) -> bool:
    if not os.path.exists(lib_path):
        return True
    t = os.path.getmtime(lib_path)
    deps = _sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, trace: bool = False) -> str:
    """Compiles every ``csrc/*.cu`` into one shared library and returns its path."""
    out = TRACE_LIB_PATH if trace else LIB_PATH
    if not force and not _stale(out):
        return out
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: the CUDA library cannot be built on this machine")
    os.makedirs(LIB_DIR, exist_ok=True)
    extra = os.environ.get("FLEXSAE_NVCC_EXTRA", "--use_fast_math").split()   # e.g. "-DFLEXSAE_BWD_MINB=8" while tuning
    if trace:
        extra = extra + ["-DFLEXSAE_TRACE"]
    tmp = f"{out}.{os.getpid()}.tmp"
    objects, log = [], ""
    try:
        running = []
        for src in _sources():                          # one compiler per source, side by side
            name = os.path.basename(src)
            flags = [f for f in extra if not (name in IEEE_SOURCES and f == "--use_fast_math")]
            obj = f"{tmp}.{name}.o"
            objects.append(obj)
            cmd = [nvcc] + NVCC_FLAGS + flags + (["-Xptxas", "-v"] if verbose else []) + ["-I", INCLUDE, "-c", "-o", obj, src]
            running.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
        done = [(p.communicate()[0], p.returncode) for p in running]
        log, failed = "".join(text for text, _ in done), any(rc for _, rc in done)
        if not failed:
            res = subprocess.run([nvcc] + NVCC_FLAGS + ["-shared", "-o", tmp] + objects, stdout=subprocess.PIPE,
                                 stderr=subprocess.STDOUT, text=True)
            log, failed = log + res.stdout, res.returncode != 0
    finally:
        for obj in objects:
            if os.path.exists(obj):
                os.remove(obj)
    if verbose or failed:
        sys.stderr.write(log)
    if failed:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError("nvcc failed:\n" + log[-4000:])
    os.replace(tmp, out)    # a reader (another rank, a running job) never sees a half-written library
    return out


def binding_path() -> str:
    """The binding is tied to the interpreter and the torch it was compiled for; both are in its name."""
    import torch

    return os.path.join(LIB_DIR, f"flexsae_binding.torch-{torch.__version__}.cp{sys.version_info[0]}{sys.version_info[1]}.so")


def build_binding(force: bool = False) -> str:
    """Compiles ``csrc/host/flexsae_binding.cpp`` against the installed torch and returns the library's path."""
    out = binding_path()
    src = os.path.join(CSRC, "host", "flexsae_binding.cpp")
    header = os.path.join(INCLUDE, "flexsae_b200.h")
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(src), os.path.getmtime(header)):
        return out
    import sysconfig

    import torch

    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found: the Python binding cannot be built on this machine")
    os.makedirs(LIB_DIR, exist_ok=True)
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [os.path.join(root, "include"), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    tmp = f"{out}.{os.getpid()}.tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    cmd += [f"-I{d}" for d in include] + [src, "-o", tmp, "-L" + os.path.join(root, "lib")]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError("g++ failed:\n" + res.stdout[-4000:])
    os.replace(tmp, out)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, trace="--trace" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
