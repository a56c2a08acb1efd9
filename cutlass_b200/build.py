"""Build ``cutlass_b200/lib/libbsgemm.so`` in-tree with nvcc for sm_100a.

Usage: ``python -m cutlass_b200.build [--force]``.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import os
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
PROFILE = os.environ.get("BSG_PROFILE") == "1"      # in-kernel timeline capture, separate file


def lib_name(profile: bool) -> str:
    return "libbsgemm" + ("_profile" if profile else "") + ".so"


OUT = os.path.join(_HERE, "lib", lib_name(PROFILE))
BINDING = os.path.join(_HERE, "lib", "_binding.so")
BINDING_STAMP = os.path.join(_HERE, "build", "binding.for")      # what it was made for
SOURCES = {      # translation unit -> the headers it includes
    "bsgemm.cu": ["gemm_kernel.cuh", "quant_kernel.cuh", "ptx.cuh", "host.h"],
    "int8.cu": ["int8_kernel.cuh", "gemm_kernel.cuh", "ptx.cuh", "host.h"],
    "activation.cu": ["activation_kernel.cuh", "int8_kernel.cuh", "gemm_kernel.cuh", "ptx.cuh", "host.h"],
    "route.cu": ["route_kernel.cuh", "gemm_kernel.cuh", "ptx.cuh", "host.h"],
}
ABI_HEADER = os.path.join("..", "..", "include", "bsgemm.h")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-cudart", "static",
]


def _objects() -> list[tuple[str, str, bool]]:
    """(source, object, is the object missing or older than what it is made from) of every translation unit."""
    out = []
    for src, headers in SOURCES.items():
        obj = os.path.join(_HERE, "build", src + (".profile" if PROFILE else "") + ".o")
        deps = [os.path.join(CSRC, f) for f in [src, ABI_HEADER] + headers]
        fresh = os.path.exists(obj) and all(os.path.getmtime(d) <= os.path.getmtime(obj) for d in deps if os.path.exists(d))
        out.append((os.path.join(CSRC, src), obj, not fresh))
    return out


def _stale() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = {os.path.join(CSRC, f) for src, headers in SOURCES.items() for f in [src, ABI_HEADER] + headers}
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _nvcc(args: list[str]) -> str:
    proc = subprocess.run([os.environ.get("NVCC", "nvcc")] + NVCC_FLAGS + args, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
    return proc.stderr


def _binding_for() -> str:
    import torch
    return f"python {sys.version_info[0]}.{sys.version_info[1]} torch {torch.__version__}"


def _compile_binding() -> None:
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DBSG_BINDING_FOR="{_binding_for()}"',
           "-isystem" + os.path.join(root, "include"), "-isystem" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem" + os.path.join(cuda, "include"), "-I" + sysconfig.get_paths()["include"], os.path.join(CSRC, "binding.cpp"), "-o", BINDING,
           "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("the compiler failed:\n" + proc.stdout + proc.stderr)


def _build_binding(force: bool) -> None:
    """The Python module of csrc/binding.cpp (host code; needs a C++ compiler, Python's and torch's headers), if it is missing, older
    than its source or made for another Python or torch.  Where it cannot be made the package works without it, so that is a
    warning."""
    deps = (os.path.join(CSRC, "binding.cpp"), os.path.join(CSRC, ABI_HEADER))
    try:
        made_for = open(BINDING_STAMP).read() if os.path.exists(BINDING_STAMP) else None
        if not force and os.path.exists(BINDING) and made_for == _binding_for() and all(os.path.getmtime(d) <= os.path.getmtime(BINDING) for d in deps):
            return
        _compile_binding()
        with open(BINDING_STAMP, "w") as f:
            f.write(_binding_for())
    except (OSError, ImportError, RuntimeError) as error:
        warnings.warn(f"the binding of the short calls was not built; they take more host time without it: {error}", RuntimeWarning)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the CUDA library, and the Python binding of its short calls, if they are missing or older than their sources;
    return the library's path.  Translation units are compiled side by side, and only those whose sources changed."""
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    os.makedirs(os.path.join(_HERE, "build"), exist_ok=True)
    if not force and not _stale():
        _build_binding(False)
        return OUT
    units = _objects()
    extra = (["-DBSG_PROFILE"] if PROFILE else []) + (["-Xptxas", "-v"] if verbose else [])
    with ThreadPoolExecutor() as pool:
        binding = pool.submit(_build_binding, force)
        logs = list(pool.map(lambda u: _nvcc(extra + ["-c", "-o", u[1], u[0]]), [u for u in units if force or u[2]]))
        binding.result()
    _nvcc(["--shared", "-o", OUT] + [u[1] for u in units])
    if verbose:
        sys.stderr.write("".join(logs))
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
