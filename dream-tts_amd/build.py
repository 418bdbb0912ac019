"""Build libdtts.so (gfx950) in-tree with hipcc.

Every ``csrc/*.hip`` compiles to an object under ``_build/`` (in parallel), then one shared
library links at ``dream-tts_amd/libdtts.so``. Where torch, its headers, Python's and g++ are there, ``csrc/serving_py.cpp``
is built against them at ``dream-tts_amd/dtts/_serving.so``, which loads the library; elsewhere ``dtts.serving`` does without.
Run as ``python dream-tts_amd/build.py``; the repository's ``__graft_entry__.build()`` calls :func:`build`.
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


def _rocm_include() -> str:
    """The headers beside the hipcc in use."""
    return os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(HIPCC) or HIPCC))), "include")


def build_binding() -> str | None:
    """``dtts/_serving.so``, or None (and a line that says what is missing) where it cannot be built; a binding of another
    build is not left in its place."""
    spec, gxx = importlib.util.find_spec("torch"), shutil.which("g++")
    python = sysconfig.get_paths()["include"]
    torch = spec.submodule_search_locations[0] if spec else ""
    missing = [what for what, there in (
        ("torch", spec), ("a ROCm torch's headers", os.path.exists(os.path.join(torch, "include", "c10", "hip", "HIPFunctions.h"))),
        ("Python.h", os.path.exists(os.path.join(python, "Python.h"))), ("g++", gxx)) if not there]
    if missing:
        if os.path.exists(BINDING):
            os.remove(BINDING)
        print(f"dtts/_serving.so is not built ({', '.join(missing)} not found): dtts.serving makes its calls from Python", file=sys.stderr)
        return None
    tmp = BINDING + ".tmp"
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",  # as torch was built
           "-isystem", os.path.join(torch, "include"), "-isystem", os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-isystem", _rocm_include(), "-isystem", python, "-I", os.path.join(REPO, "include"),
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
