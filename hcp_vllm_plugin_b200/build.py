"""Build ``libhcp_ring.so`` in-tree with nvcc for sm_100a, and ``_hcp_front.so``.

    python -m hcp_vllm_plugin_b200.build

The library links the CUDA runtime statically and resolves the driver's
``cuTensorMapEncodeTiled`` at run time, so it loads on any box with the
NVIDIA driver and needs no torch at link time.  ``_hcp_front.so`` is the
torch front end of the serving-step entry points (``csrc/front.cpp``, no
kernels): an extension module for the installed torch and Python, left out
where there is no torch.
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libhcp_ring.so")
SOURCES = [os.path.join(CSRC, "hcp_ring.cu")]
HEADER = os.path.join(ROOT, "include", "hcp_ring.h")
DEPS = SOURCES + sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + [HEADER]
FRONT = os.path.join(HERE, "_hcp_front.so")
FRONT_SOURCE = os.path.join(CSRC, "front.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = os.path.join(cuda_home, "bin", "nvcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found (set CUDA_HOME)")
    return found


def up_to_date(target: str | None = None, deps=DEPS) -> bool:
    target = LIB if target is None else target
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps if os.path.exists(d))


def _compile(cmd: list[str], target: str, verbose: bool) -> None:
    tmp = target + ".tmp"
    cmd = [tmp if c == target else c for c in cmd]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, target)


def front_target() -> str:
    """What the front end has to be built for; the module carries it (``built_for``)."""
    import torch

    return (f"torch {torch.__version__}, C++ ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"Python {sys.version_info.major}.{sys.version_info.minor} {sysconfig.get_config_var('SOABI')}")


def _front_is_current() -> bool:
    if not up_to_date(FRONT, [FRONT_SOURCE, HEADER]):
        return False
    with open(FRONT, "rb") as f:
        return front_target().encode() in f.read()


def build_front(force: bool = False, verbose: bool = False) -> str:
    """Compile the torch front end with the host compiler."""
    if not force and _front_is_current():
        return FRONT
    import torch

    home = os.path.dirname(torch.__file__)
    # of the toolkit the headers alone: no runtime library of it is linked
    includes = [os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"),
                os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include"), sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DHCP_BUILT_FOR="{front_target()}"', "-I", os.path.join(ROOT, "include"),
           *(a for p in includes for a in ("-isystem", p)), "-o", FRONT, FRONT_SOURCE,
           "-L", os.path.join(home, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
           "-ltorch_python"]
    _compile(cmd, FRONT, verbose)
    return FRONT


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        cmd = [nvcc_path(), *NVCC_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-o", LIB, *SOURCES]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        _compile(cmd, LIB, verbose)
    try:
        import torch  # noqa: F401
    except ImportError as e:  # a host of the C ABI alone
        print(f"{FRONT} is not built: it is the front end for torch, which cannot be imported ({e})", file=sys.stderr)
    else:
        build_front(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
