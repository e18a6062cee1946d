"""In-tree build of the native library.

    python -m elasticmegatron_amd.build

Compiles csrc/*.hip for gfx950 into csrc/libemrs.so with hipcc.
"""

import glob
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(CSRC, "libemrs.so")

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-amdgpu-kernarg-preload-count=14",  # leading kernel arguments arrive in scalar registers
    "-Wall", "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found")


def build_native(verbose: bool = False) -> str:
    """Each source compiles in a process of its own, as many at once as there are CPUs (at most 8)."""
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    logs = []
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in srcs]

        def compile_one(src_obj):
            src, obj = src_obj
            return subprocess.run([hipcc(), *flags, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-c", src, "-o", obj],
                                  capture_output=True, text=True)

        with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
            logs += pool.map(compile_one, zip(srcs, objs))
        out = LIB + ".tmp"
        if all(r.returncode == 0 for r in logs):
            logs.append(subprocess.run([hipcc(), *HIPCC_FLAGS, *objs, "-o", out], capture_output=True, text=True))
    failed = [r for r in logs if r.returncode != 0]
    if failed:
        raise RuntimeError("hipcc failed:\n" + "".join(r.stdout + r.stderr for r in failed))
    if verbose:
        noise = "is not a recognized feature for this target"
        print("\n".join(l for r in logs for l in (r.stdout + r.stderr).splitlines() if noise not in l))
    os.replace(out, LIB)
    return LIB


def main() -> int:
    print(build_native(verbose=True))
    return 0


if __name__ == "__main__":
    sys.exit(main())
