"""In-tree build of the native libraries (no cmake, no JIT cache):

* ``libpvae_prep.so``  g++   host-only genotype front end (csrc/pvae_prep.cpp)
* ``libpvae.so``       hipcc --offload-arch=gfx950   HIP kernels + engine + C ABI (csrc/pvae_engine.hip) and the
                       operators on device tensors (csrc/pvae_ops.hip)

Both land next to this file so that they travel to the GPU box with the source snapshot.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INC = os.path.join(os.path.dirname(HERE), "include")


def _newer(target, sources):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _run(cmd):
    print("+", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def build_prep(force=False):
    out = os.path.join(HERE, "libpvae_prep.so")
    srcs = [os.path.join(CSRC, "pvae_prep.cpp"), os.path.join(INC, "pvae_prep.h")]
    if force or _newer(out, srcs):
        _run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-o", out, srcs[0], "-lz"])
    return out


def build_engine(force=False, extra=()):
    out = os.path.join(HERE, "libpvae.so")
    srcs = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".hip", ".h", ".hpp"))]
    srcs += [os.path.join(INC, "pvae.h"), os.path.join(INC, "pvae_ops.h")]
    if force or _newer(out, srcs):
        hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
        # no packed float32 instructions: some of their forms have given wrong results on this part (the host pass of hipcc does
        # not know the feature and says so)
        flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-Wno-unused-value",
                 "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", *extra]
        with tempfile.TemporaryDirectory() as tmp:
            objs, running = [], []
            for name in ("pvae_engine", "pvae_ops"):
                objs.append(os.path.join(tmp, name + ".o"))
                cmd = [hipcc, *flags, "-c", "-o", objs[-1], os.path.join(CSRC, name + ".hip")]
                print("+", " ".join(cmd), flush=True)
                running.append((cmd, subprocess.Popen(cmd)))
            for cmd, p in running:
                if p.wait():
                    raise subprocess.CalledProcessError(p.returncode, cmd)
            _run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", out, *objs])
    return out


def build_all(force=False):
    return build_prep(force), build_engine(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
