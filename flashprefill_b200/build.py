"""Builds libflashprefill_b200.so (sm_100a) in-tree with nvcc.

    python -m flashprefill_b200.build [--verbose-ptxas]

The library is one unity translation unit (csrc/fp_api.cu includes the kernels) linked
against the static CUDA runtime, so it only needs the NVIDIA driver at run time.  Behind it
_fp_torch.so (csrc/fp_torch.cpp, g++) is built, which passes torch tensors to the paged-cache entry
points; it goes by the torch that it was built for, and C callers do not need it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libflashprefill_b200.so")
SOURCES = ["fp_api.cu"]
EXT = os.path.join(HERE, "_fp_torch.so")
EXT_TAG = EXT + ".built_for"
EXT_SOURCE = "fp_torch.cpp"
HEADER = os.path.join(os.path.dirname(HERE), "include", "flashprefill_b200.h")


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the CUDA toolkit is needed to build flashprefill_b200")


def _deps():
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))]
    deps.append(HEADER)
    return deps


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for d in _deps())


def _ext_tag() -> str:
    """What _fp_torch.so depends on beside its source: torch's C++ interface and Python's."""
    import sysconfig

    import torch
    return f"{torch.__version__} {sysconfig.get_config_var('SOABI')}"


def ext_needs_build() -> bool:
    src = os.path.join(CSRC, EXT_SOURCE)
    if not (os.path.exists(EXT) and os.path.exists(EXT_TAG)):
        return True
    if any(os.path.getmtime(d) >= os.path.getmtime(EXT) for d in (src, HEADER)):
        return True
    with open(EXT_TAG) as f:
        return f.read() != _ext_tag()


def build_ext(force: bool = False) -> str:
    """_fp_torch.so: plain g++ against torch's headers (its C++ interface has no device code)."""
    if not force and not ext_needs_build():
        return EXT
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    src = os.path.join(CSRC, EXT_SOURCE)
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DFPB_BUILT_FOR="{torch.__version__}"',
           "-o", EXT + ".tmp", src]
    for d in cpp_extension.include_paths() + [sysconfig.get_paths()["include"], os.path.join(cuda, "include")]:
        cmd += ["-isystem", d]
    for d in cpp_extension.library_paths():
        cmd += ["-L" + d]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    os.replace(EXT + ".tmp", EXT)
    with open(EXT_TAG, "w") as f:
        f.write(_ext_tag())
    return EXT


def build(force: bool = False, ptxas_verbose: bool = False) -> str:
    lib = build_lib(force, ptxas_verbose)  # first: it needs neither g++ nor torch's headers
    build_ext(force)
    return lib


def build_lib(force: bool = False, ptxas_verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    cmd = [nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
           "-shared", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
           "-cudart", "static", "-o", LIB + ".tmp"]
    if ptxas_verbose:
        cmd += ["-Xptxas", "-v"]
    # extra nvcc flags, e.g. -DFPB_SA_PROFILE=1 for an instrumented build
    cmd += os.environ.get("FLASHPREFILL_B200_NVCC_FLAGS", "").split()
    cmd += [os.path.join(CSRC, s) for s in SOURCES]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    if ptxas_verbose:
        sys.stderr.write(r.stderr)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force=True, ptxas_verbose="--verbose-ptxas" in sys.argv))
