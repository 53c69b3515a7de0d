"""Build libsabre_b200.so in-tree with nvcc for sm_100a, and with the host compiler
the extension that calls its paged entry points from torch (_paged_call.so).

    python -m sabrecoder_b200.build          # build if sources changed
    python -m sabrecoder_b200.build --force  # always rebuild
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libsabre_b200.so")
CALL = os.path.join(PKG, "_paged_call.so")
CALL_SOURCE = os.path.join(CSRC, "paged_call.cpp")
HEADER = os.path.join(ROOT, "include", "sabre_b200.h")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-shared",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) + [HEADER])


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(s) <= t for s in sources())


def _run(cmd, tmp: str, out: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, out)


def build_call(force: bool = False, verbose: bool = False) -> str:
    """The torch extension; linked to libsabre_b200.so beside it. It holds torch's and
    Python's ABI, so the file beside it says which ones it was built for."""
    import sysconfig

    import torch
    stamp = CALL + ".for"
    key = f"torch {torch.__version__} python {sys.version}"
    if not force and os.path.exists(CALL) and os.path.exists(stamp):
        with open(stamp) as f:
            same = f.read() == key
        if same and all(os.path.getmtime(f) <= os.path.getmtime(CALL) for f in (CALL_SOURCE, HEADER)):
            return CALL
    home = os.path.dirname(torch.__file__)
    inc = [os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    tmp = CALL + ".tmp"
    _run([os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in inc), CALL_SOURCE,
          "-o", tmp, f"-L{PKG}", "-l:" + os.path.basename(LIB), f"-L{os.path.join(home, 'lib')}", "-lc10",
          "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"],
         tmp, CALL, verbose)
    with open(stamp, "w") as f:
        f.write(key)
    return CALL


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        tmp = LIB + ".tmp"
        _run([nvcc(), *NVCC_FLAGS, "-o", tmp, os.path.join(CSRC, "sabre_capi.cu")], tmp, LIB, verbose)
    build_call(force, verbose)
    return LIB


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args(argv)
    print(build(force=a.force, verbose=True))


if __name__ == "__main__":
    sys.exit(main())
