"""Build the CUDA library in-tree: ``python bioemu2_b200/build.py`` (or ``python __graft_entry__.py``).

One nvcc invocation compiles ``csrc/lib.cu`` (which includes every kernel) for sm_100a into
``libb200pair.so`` beside this file, and one of the host compiler ``csrc/training_binding.cpp`` into the extension module
``_training.so`` (against torch's headers; what it was built for stands in ``_training.so.for`` beside it, and another torch or Python
builds it anew).  nvcc cross-compiles, so no GPU is needed to build.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libb200pair.so")
SRC = os.path.join(HERE, "csrc", "lib.cu")
BINDING_PATH = os.path.join(HERE, "_training.so")
BINDING_SRC = os.path.join(HERE, "csrc", "training_binding.cpp")
BINDING_FOR = BINDING_PATH + ".for"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
]


def sources() -> list[str]:
    csrc = os.path.join(HERE, "csrc")
    return [os.path.join(csrc, f) for f in sorted(os.listdir(csrc)) if f.endswith((".cu", ".cuh", ".inc"))] + headers()


def headers() -> list[str]:
    inc = os.path.join(os.path.dirname(HERE), "include")
    return [os.path.join(inc, f) for f in sorted(os.listdir(inc)) if f.endswith(".h")]


def is_stale(path: str = LIB_PATH, of: list[str] | None = None) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(s) > t for s in of or sources())


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed:\n{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stderr)


def build_library(verbose: bool = False) -> None:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    _run([nvcc, *(["-Xptxas=-v"] if verbose else []), *NVCC_FLAGS, "-o", LIB_PATH, SRC], verbose)


def binding_for() -> str:
    """The Python and the torch that an extension built now would be for."""
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    with open(os.path.join(torch, "version.py")) as version:
        return f"{sysconfig.get_config_var('SOABI')}\n{version.read()}"


def binding_is_stale() -> bool:
    if is_stale(BINDING_PATH, [BINDING_SRC, *headers()]) or not os.path.exists(BINDING_FOR):
        return True
    with open(BINDING_FOR) as known:
        return known.read() != binding_for()


def build_binding(verbose: bool = False) -> None:
    from torch import compiled_with_cxx11_abi

    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    includes = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"), cuda,
                sysconfig.get_paths()["include"]]
    _run([shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(compiled_with_cxx11_abi())}",
          *(f"-I{i}" for i in includes), BINDING_SRC, "-o", BINDING_PATH, "-L" + os.path.join(torch, "lib"), "-ltorch_python", "-ltorch_cpu",
          "-lc10", "-lc10_cuda"], verbose)
    with open(BINDING_FOR, "w") as known:
        known.write(binding_for())


def build(force: bool = False, verbose: bool = False) -> str:
    wanted = [f for f, stale in ((build_library, is_stale), (build_binding, binding_is_stale)) if force or stale()]
    with ThreadPoolExecutor(2) as pool:  # two compilers, neither of which waits for the other
        for done in [pool.submit(f, verbose) for f in wanted]:
            done.result()
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
