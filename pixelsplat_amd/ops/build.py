"""Builds libpixelsplat_ops.so in-tree with hipcc for gfx950 (cross-compiles without a GPU), and _binding.so, the
operators as torch functions over it, with the host's compiler.

    python -m pixelsplat_amd.ops.build [--force] [--verbose]

A library of its own next to libpixelsplat_hip.so: the counters and test logs committed for the rasterizer and the
epipolar kernels are tied to the hashes of that library's sources, which these operators do not change.
"""
from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import sysconfig

from ..build import _hipcc

HERE = os.path.dirname(os.path.abspath(__file__))
PACKAGE = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(PACKAGE, "libpixelsplat_ops.so")
BINDING = os.path.join(HERE, "_binding.so")
HEADERS = [os.path.join(HERE, "include", "pixelsplat_ops.h"),
           os.path.join(os.path.dirname(PACKAGE), "include", "pixelsplat_hip.h")]
INFO_UNIT = "ops_info.hip"      # carries every unit's hash (ps_ops_build_info)

# -packed-fp32-ops: fp32 code stays scalar.  The compiler pairs ordinary float code into packed instructions by
# itself, and results are not to depend on which of their forms it picks.
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def units() -> list[str]:
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def unit_hashes() -> str:
    """"<file>:<hash12> ..." -- per translation unit, sha256 over the headers, its source and the flags."""
    shared = hashlib.sha256(" ".join(FLAGS).encode())
    for h in [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".h")] + HEADERS:
        shared.update(open(h, "rb").read())
    out = []
    for name in units():
        h = shared.copy()
        h.update(open(os.path.join(CSRC, name), "rb").read())
        out.append(f"{name[:-4]}:{h.hexdigest()[:12]}")
    return " ".join(out)


def build(force: bool = False, verbose: bool = False) -> str:
    hashes = unit_hashes()
    want = dict(tok.split(":") for tok in hashes.split())
    include = ["-I", CSRC] + [x for h in HEADERS for x in ("-I", os.path.dirname(h))]
    objs, procs = [], []
    for name in units():
        src, obj = os.path.join(CSRC, name), os.path.join(CSRC, name[:-4] + ".o")
        flags = [*FLAGS, *include]
        stamp = want[name[:-4]]
        if name == INFO_UNIT:
            flags.append(f'-DPS_BUILD_HASHES="{hashes}"')
            stamp = hashlib.sha256(hashes.encode()).hexdigest()[:12]
        objs.append(obj)
        mark = obj + ".tmp"                 # the hash that the object was built from
        if not force and os.path.exists(obj) and os.path.exists(mark) and open(mark).read() == stamp:
            continue
        cmd = [_hipcc(), *flags, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((name, mark, stamp, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                                          text=True)))
    failed = []
    for name, mark, stamp, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"hipcc failed on {name}:\n{out}")
            continue
        with open(mark, "w") as f:
            f.write(stamp)
        if verbose and out.strip():
            print(out)
    if failed:
        raise RuntimeError("\n".join(failed))
    if procs or not os.path.exists(LIB):
        subprocess.check_call([_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", LIB])
    build_binding(force, verbose)
    return LIB


def build_binding(force: bool = False, verbose: bool = False) -> str:
    import torch
    from torch.utils import cpp_extension

    src = os.path.join(CSRC, "binding.cpp")
    flags = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__"]
    stamp = hashlib.sha256(" ".join([*flags, torch.__version__, sys.version]).encode())
    for path in [src, *HEADERS]:
        stamp.update(open(path, "rb").read())
    mark = os.path.join(CSRC, "binding.o.tmp")
    if not force and os.path.exists(BINDING) and os.path.exists(mark) and open(mark).read() == stamp.hexdigest():
        return BINDING
    cmd = ["g++", *flags, src, "-o", BINDING]
    cmd += [x for h in HEADERS for x in ("-I", os.path.dirname(h))]
    cmd += [x for d in [*cpp_extension.include_paths(), "/opt/rocm/include", sysconfig.get_paths()["include"]]
            for x in ("-isystem", d)]
    cmd += [x for d in cpp_extension.library_paths() for x in ("-L", d)] + ["-L", PACKAGE]
    cmd += ["-lpixelsplat_ops", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_python", "-Wl,-rpath,$ORIGIN/.."]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on binding.cpp:\n{r.stdout}")
    with open(mark, "w") as f:
        f.write(stamp.hexdigest())
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv or "-v" in sys.argv))
