"""Build libwm.so (gfx950 HIP kernels + C ABI) in-tree with hipcc.  No GPU needed to compile."""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libwm.so")
ARCH = "gfx950"
# No v_pk_{add,mul,fma}_f32: hipcc -O3 forms them from ordinary float code, and some of their forms have
# given wrong results on this hardware now and then.  (The host pass warns that it does not know the
# feature.)  The older sources keep the code they were validated with: without the packed forms their
# float contraction changes, and kernels that are tested to agree bit for bit no longer do.
NO_PACKED_F32 = ("-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops")
SCALAR_F32_SOURCES = {"dropout.hip", "grouped.hip", "int8.hip"}
# Accumulators of matrix instructions in ordinary registers: in the accumulator file the tile loops of these
# sources carried 100 register moves for 32 matrix instructions.
VGPR_FORM = ("-mllvm", "-amdgpu-mfma-vgpr-form=1")
VGPR_FORM_SOURCES = {"grouped.hip", "int8.hip"}


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found (need ROCm to build libwm.so)")
    return exe


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, extra=()):
    obj = os.path.join(OBJ, src[:-4] + ".o")
    deps = [os.path.join(CSRC, src), os.path.join(ROOT, "include", "wm.h")] + \
        [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".h")]
    if not _stale(obj, deps):
        return obj
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall",
           "-Wno-unused-function", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
           "-I", "/opt/rocm/include",
           *(NO_PACKED_F32 if src in SCALAR_F32_SOURCES else ()),
           *(VGPR_FORM if src in VGPR_FORM_SOURCES else ()), *extra, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if r.stderr.strip():
        sys.stderr.write(r.stderr)
    return obj


def build(force: bool = False, jobs: int = 4) -> str:
    os.makedirs(OBJ, exist_ok=True)
    if force:
        for f in os.listdir(OBJ):
            os.remove(os.path.join(OBJ, f))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, sources()))
    if force or _stale(LIB, objs):
        cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", LIB, *objs, "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
