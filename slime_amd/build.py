"""Builds ``slime_amd/libslime_ca.so`` (the HIP kernels + C ABI) for gfx950, and
``slime_amd/libslime_probe.so`` (the ceiling measurements of ``calibrate.py``), and
``slime_amd/_binding.so`` (the attention calls over torch tensors, host code; left out where no
torch for ROCm is installed, since the library does not need it).

Each source is compiled with hipcc in parallel into ``slime_amd/_build/`` and
linked into one shared library next to this file. Packed-fp32 instructions are
disabled for all device code (``-Xclang -target-feature -Xclang
-packed-fp32-ops``).

Usage: ``python -m slime_amd.build`` (also called by ``__graft_entry__.build``).
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libslime_ca.so")
PROBE_LIB = os.path.join(HERE, "libslime_probe.so")  # measured ceilings (calibrate.py)
BINDING = os.path.join(HERE, "_binding.so")  # attention.py's calls over torch tensors
SOURCES = ["api.cpp", "gemm.hip", "gemm_small.hip", "gemm_add.hip", "gemm_tape.hip", "stencil.hip", "mass.hip", "fitness.hip", "organism.hip",
           "backward.hip", "pool.hip", "head_norm.hip", "attend.hip", "attend_backward.hip"]
ARCH = "gfx950"


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found; the HIP library cannot be built")


def flags() -> list:
    return [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall",
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            f"-I{os.path.join(os.path.dirname(HERE), 'include')}"]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    cmd = [hipcc(), *flags(), "-x", "hip", "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def _torch_folder():
    """Where a torch for ROCm is installed, or None: a C or C++ host needs the library alone."""
    spec = importlib.util.find_spec("torch")
    folder = list(spec.submodule_search_locations)[0] if spec and spec.submodule_search_locations else None
    return folder if folder and os.path.exists(os.path.join(folder, "lib", "libc10_hip.so")) else None


def _build_binding(torch: str) -> None:
    """The CPython module (host code only), against torch's headers and the library just linked. It
    holds torch's version, which attention.load compares with the running one's."""
    with open(os.path.join(torch, "version.py")) as f:
        version = re.search(r"^__version__\s*=\s*['\"](.+?)['\"]", f.read(), re.M).group(1)
    tmp = BINDING + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f'-DSLIME_TORCH="{version}"', f"-I{os.path.join(os.path.dirname(HERE), 'include')}", f"-I{torch}/include",
           f"-I{torch}/include/torch/csrc/api/include", f"-I{sysconfig.get_path('include')}",
           f"-isystem{os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc()))), 'include')}",
           os.path.join(CSRC, "binding.cpp"), f"-L{HERE}", "-l:libslime_ca.so", "-Wl,-rpath,$ORIGIN",
           f"-L{torch}/lib", "-lc10", "-ltorch_cpu", "-ltorch_python", "-lc10_hip", "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"build of binding.cpp failed:\n{r.stderr}")
    os.replace(tmp, BINDING)


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    tmp = PROBE_LIB + ".tmp"
    cmd = [hipcc(), *flags(), "-x", "hip", "-shared", os.path.join(CSRC, "probe.hip"), "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for probe.hip:\n{r.stderr}")
    os.replace(tmp, PROBE_LIB)
    torch = _torch_folder()
    if torch:
        _build_binding(torch)
    if verbose:
        print(f"built {LIB} and {PROBE_LIB}" + (f" and {BINDING}" if torch else "; no torch for ROCm here, so no "
                                                f"{BINDING}: slime_amd.attend and its like will raise"))
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
