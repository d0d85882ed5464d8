"""Build recipe for ``lich_amd/libipc_hip.so`` (gfx950 only).

Every ``csrc/*.hip`` file is compiled by ``hipcc --offload-arch=gfx950`` into
an object in ``lich_amd/_build/`` (in parallel) and linked into the shared
library next to this file, so that the built library travels with the source
tree.  No torch headers are used there: the boundary is the plain C ABI of
``include/ipc_hip.h``.  ``csrc/ipc_fast_call.cpp`` (host code: the microscaled calls'
checks and arguments without Python's overhead) is compiled against torch's headers
into ``lich_amd/_fast_call.so``.

Run ``python -m lich_amd.build`` (or ``__graft_entry__.build()``).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libipc_hip.so"
ARCH = "gfx950"

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

COMMON = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-mcode-object-version=5",
    # Packed-fp32 VALU forms are kept out of every kernel (see module docstring of ipc_device.h).
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-result",
    "-Wno-unused-variable",
]


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [HIPCC, *COMMON, "-I", str(PKG.parent / "include"), "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    # The host pass does not know the packed-fp32 feature; that warning is expected.
    noise = [ln for ln in res.stderr.splitlines() if "packed-fp32-ops" not in ln and ln.strip()]
    if noise and verbose:
        print("\n".join(noise), flush=True)
    return obj


def _extension(verbose: bool) -> Path:
    import torch

    at, out = Path(torch.__file__).parent, PKG / "_fast_call.so"
    tmp = out.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-isystem", str(at / "include"),
           "-I", sysconfig.get_paths()["include"], str(CSRC / "ipc_fast_call.cpp"), "-o", str(tmp),
           "-L", str(at / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for ipc_fast_call.cpp:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    return out


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile every HIP source and link ``libipc_hip.so``, and the extension; returns the library's path."""
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(sources), max(1, (os.cpu_count() or 2)), 8)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        extension = ex.submit(_extension, verbose)
        objs = list(ex.map(lambda s: _compile(s, verbose), sources))
        extension.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv)
    print(path)
