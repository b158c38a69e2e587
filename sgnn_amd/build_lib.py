"""Build libsgnn_hip.so in-tree with hipcc for gfx950 (no JIT cache: the .so
travels to the GPU box with the repo snapshot)."""
from __future__ import annotations

import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "_lib")
LIB = os.path.join(LIBDIR, "libsgnn_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-shared",
         "-ffp-contract=fast", "-munsafe-fp-atomics", "-Wno-unused-result",
         # no packed fp32 instructions: some of their forms have given wrong results now and then (the host pass
         # says that it does not know the feature)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# the radius search's translation unit without FMA contraction: its graphs are bit-exact against the
# oracle's `dims summed in order, no contraction` rule (the distance blocks of the other units carry
# `#pragma clang fp contract(off)` as well)
NO_CONTRACT = {"radius.hip"}


def flags_for(src: str):
    f = [x for x in FLAGS if x != "-shared"]
    if os.path.basename(src) in NO_CONTRACT:
        f = ["-ffp-contract=off" if x == "-ffp-contract=fast" else x for x in f]
    return f


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def deps():
    return sources() + glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(ROOT, "include", "sgnn.h")]


def needs_build() -> bool:
    if not (os.path.exists(LIB) and os.path.exists(TORCH_OPS)):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for d in deps()) or torch_ops_stale()


# the torch binding of the typed operators (host code alone; opens libsgnn_hip.so at run time)
TORCH_OPS_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_OPS = os.path.join(LIBDIR, "_torch_ops.so")


def torch_ops_stale() -> bool:
    return not os.path.exists(TORCH_OPS) or any(
        os.path.getmtime(f) > os.path.getmtime(TORCH_OPS)
        for f in (TORCH_OPS_SRC, os.path.join(ROOT, "include", "sgnn.h"), __file__))


def start_torch_ops() -> subprocess.Popen:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(HIPCC))) if os.path.exists(HIPCC) else "/opt/rocm"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in (*include_paths(), os.path.join(rocm, "include"), sysconfig.get_paths()["include"])],
           TORCH_OPS_SRC, "-o", TORCH_OPS + ".tmp", f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10",
           "-lc10_hip", "-ldl"]
    return subprocess.Popen(cmd)


OBJDIR = os.path.join(LIBDIR, "obj")   # per-source objects (git- and gpurun-ignored): incremental rebuilds


def build(force: bool = False, verbose: bool = False, defines=(), lib: str = LIB) -> str:
    """Compile every csrc/*.hip for gfx950 and link `lib`.  `defines` (e.g.
    SGNN_PROBE) are for experiment builds linked to another path.  A source is
    recompiled when it, any header, or this script is newer than its object."""
    if not force and not defines and lib == LIB and not needs_build():
        return LIB
    os.makedirs(OBJDIR, exist_ok=True)
    objs = []
    procs = []
    tag = "".join("_" + d.lower().replace("=", "_") for d in defines)
    headers = glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(ROOT, "include", "sgnn.h"), __file__]
    newest_header = max(os.path.getmtime(h) for h in headers)
    for src in sources():
        obj = os.path.join(OBJDIR, os.path.basename(src) + tag + ".o")
        objs.append(obj)
        if (not force and os.path.exists(obj) and os.path.getmtime(obj) > os.path.getmtime(src)
                and os.path.getmtime(obj) > newest_header):
            continue
        cmd = [HIPCC, *flags_for(src), *[f"-D{d}" for d in defines], "-c", src, "-o", obj + ".tmp",
               "-I", os.path.join(ROOT, "include")]
        if verbose:
            print(" ".join(cmd))
        procs.append((subprocess.Popen(cmd), obj))
    if lib == LIB and (force or torch_ops_stale()):
        if start_torch_ops().wait() != 0:
            raise RuntimeError("building the torch binding failed")
        os.replace(TORCH_OPS + ".tmp", TORCH_OPS)
    for p, obj in procs:
        if p.wait() != 0:
            raise RuntimeError("hipcc failed")
        os.replace(obj + ".tmp", obj)
    tmp = lib + ".tmp"
    subprocess.check_call([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs])
    os.replace(tmp, lib)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
