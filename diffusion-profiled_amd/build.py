"""Build the gfx950 HIP library ``lib/libdpa_fp8.so`` from ``csrc/*.hip``.

The library has a plain C ABI (``include/dpa_fp8.h``) and does not link against torch.
Sources compile in parallel (one ``hipcc -c`` per file) and link with ``hipcc -shared``. Beside it
``lib/dpa_fast_calls.so`` (``csrc/fast_calls.cpp``, host code only) is a Python module for the torch
of this interpreter; without torch, its headers or g++ the library is built alone, with a warning, and the
module's calls take the general way through Python.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
import warnings
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC_DIR = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_DIR = PKG_DIR / "lib"
LIB_PATH = LIB_DIR / "libdpa_fp8.so"
FAST_PATH = LIB_DIR / "dpa_fast_calls.so"

OFFLOAD_ARCH = "gfx950"

# -ffp-contract=off keeps every fp32 rounding step of the reference recipe explicit; the
# packed-fp32 target feature is switched off for all device code.
HIPCC_FLAGS = [
    f"--offload-arch={OFFLOAD_ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    path = shutil.which("hipcc") or os.path.join(rocm, "bin", "hipcc")
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found; the FP8 HIP library cannot be built")
    return path


def sources() -> list[Path]:
    return sorted(CSRC_DIR.glob("*.hip"))


def _fast_calls_command() -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
            "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include",
            f"-I{sysconfig.get_paths()['include']}", f"-I{rocm}/include",
            str(CSRC_DIR / "fast_calls.cpp"), "-o", str(FAST_PATH.with_suffix(".so.tmp")),
            f"-L{root}/lib", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]


def build_library(verbose: bool = False) -> Path:
    """Compile every csrc/*.hip for gfx950 and link lib/libdpa_fp8.so. Always rebuilds."""
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    cc = hipcc()
    procs = []
    objs = []
    for src in sources():
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        cmd = [cc, *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    fast, why = None, ""
    try:
        fast = subprocess.Popen(_fast_calls_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    except (ImportError, OSError) as e:     # no torch, no g++
        why = str(e)
    errors = []
    for src, p in procs:
        out, _ = p.communicate()
        text = out.decode(errors="replace")
        # the host pass warns that it does not know the packed-fp32 feature: harmless
        lines = [ln for ln in text.splitlines() if "packed-fp32-ops" not in ln and ln.strip()]
        if p.returncode != 0:
            errors.append(f"{src.name}:\n" + "\n".join(lines))
        elif verbose and lines:
            print("\n".join(lines), flush=True)
    if fast is not None:
        out, _ = fast.communicate()
        why = out.decode(errors="replace") if fast.returncode != 0 else ""
    if errors:
        raise RuntimeError("hipcc failed:\n" + "\n\n".join(errors))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [cc, f"--offload-arch={OFFLOAD_ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError("hipcc link failed:\n" + r.stdout.decode(errors="replace"))
    os.replace(tmp, LIB_PATH)
    if why:
        FAST_PATH.unlink(missing_ok=True)       # (one of another build would not fit this library)
        warnings.warn(f"{FAST_PATH.name} was not built, its calls go through Python: {why}")
    else:
        os.replace(FAST_PATH.with_suffix(".so.tmp"), FAST_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(verbose=True))
