"""Build libdtts.so (gfx950) in-tree with hipcc.

Every ``csrc/*.hip`` compiles to an object under ``_build/`` (in parallel), then one shared
library links at ``dream-tts_amd/libdtts.so``, and ``csrc/serving_py.cpp`` (host code against torch's
and Python's headers) at ``dream-tts_amd/dtts/_serving.so``, which loads it. Run as ``python dream-tts_amd/build.py``; the
repository's ``__graft_entry__.build()`` calls :func:`build`.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libdtts.so")
BINDING = os.path.join(HERE, "dtts", "_serving.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# -packed-fp32-ops: keep the compiler from emitting v_pk_{add,mul,fma}_f32.
COMMON = [
    "-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950", "-mcode-object-version=5",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unknown-pragmas",
    "-I", os.path.join(REPO, "include"), "-I", CSRC,
]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src)[:-4] + ".o")
    cmd = [HIPCC, *COMMON, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    # the host pass does not know the packed-fp32 feature and says so; anything else is shown
    noise = "is not a recognized feature for this target"
    msg = "\n".join(l for l in (r.stderr or "").splitlines() if noise not in l and "(ignoring feature)" not in l)
    if msg.strip():
        print(msg, file=sys.stderr)
    return obj


def build(jobs: int | None = None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4, 16)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    shutil.move(tmp, LIB)
    build_binding()
    return LIB


def build_binding() -> str:
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    tmp = BINDING + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",  # as torch was built
           "-isystem", os.path.join(torch, "include"), "-isystem", os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-isystem", "/opt/rocm/include", "-isystem", sysconfig.get_paths()["include"], "-I", os.path.join(REPO, "include"),
           os.path.join(CSRC, "serving_py.cpp"), "-o", tmp,
           "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python",
           "-L" + HERE, "-l:libdtts.so", "-Wl,-rpath,$ORIGIN/.."]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"binding failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    shutil.move(tmp, BINDING)
    return BINDING


if __name__ == "__main__":
    print(build())
