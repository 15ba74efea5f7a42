#!/usr/bin/env python3
"""Build libuniter_hip.so (gfx950) in-tree with hipcc, and uniter_nodes.so (nodes.cpp: host code, autograd nodes) with g++.

    python uniter_amd/csrc/build.py [--force] [--verbose]

One object per .hip file (parallel), linked into uniter_amd/csrc/build/libuniter_hip.so.  Rebuilds only
objects whose sources (or the headers they include) are newer.  hipcc cross-compiles without a GPU.
"""
import argparse
import concurrent.futures as cf
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
# (variant builds for A/B runs: UNITER_BUILD_DIR=build_b UNITER_EXTRA_FLAGS="-DUNITER_STORE_POLICY=2" python build.py; a process picks
#  a variant up through UNITER_AMD_LIB=<path to its libuniter_hip.so> / LD_LIBRARY_PATH for the native harness)
BUILD = os.path.join(HERE, os.environ.get("UNITER_BUILD_DIR", "build"))
LIB = os.path.join(BUILD, "libuniter_hip.so")
NODES = os.path.join(BUILD, "uniter_nodes.so")
SOURCES = ["capi.hip", "gemm.hip", "attention.hip", "layernorm.hip", "embed.hip", "adamw.hip", "encoder.hip", "comm.hip", "ot.hip", "pool.hip", "lmhead.hip", "head.hip", "rotary.hip",
           "diff_attention.hip"]
ARCH = "gfx950"
# No packed FP32 arithmetic (v_pk_add / mul / fma_f32) in device code: some of its forms have given wrong results now and then, with no
# error, and -O3 forms it by itself from ordinary float code.  (The host pass does not know the feature and warns: harmless.)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def find_hipcc():
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _sources_of(path, seen=None):
    """`path`, the files that it includes by name (recursively) and this script, whose flags they are compiled with."""
    seen = {os.path.abspath(__file__)} if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen:
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', f.read(), flags=re.M):
                _sources_of(os.path.join(os.path.dirname(path), name), seen)
    return seen


def build_nodes(force=False, verbose=False):
    """nodes.cpp against the torch that is installed (found without importing it).  It links no part of libuniter_hip.so."""
    src = os.path.join(HERE, "nodes.cpp")
    if not force and not _stale(NODES, _sources_of(src)):
        return NODES
    os.makedirs(BUILD, exist_ok=True)
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    inc = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D_GLIBCXX_USE_CXX11_ABI=1", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-DTORCH_EXTENSION_NAME=uniter_nodes"]
    for d in inc:
        cmd += ["-isystem", d]
    cmd += [src, "-o", NODES, "-L" + os.path.join(torch, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed on %s" % src)
    return NODES


def build(force=False, verbose=False):
    hipcc = find_hipcc()
    os.makedirs(BUILD, exist_ok=True)
    flags = ["--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "-Wall", "-Wno-unused-function",
             "-DNDEBUG"] + NO_PACKED_FP32 + os.environ.get("UNITER_EXTRA_FLAGS", "").split()
    jobs = []
    objs = []
    for src in SOURCES:
        s = os.path.join(HERE, src)
        o = os.path.join(BUILD, src.replace(".hip", ".o"))
        objs.append(o)
        if force or _stale(o, _sources_of(s)):
            jobs.append((s, o))

    def compile_one(job):
        s, o = job
        cmd = [hipcc] + flags + ["-c", s, "-o", o]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        return s, r

    with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs) + 1)) as ex:
        nodes = ex.submit(build_nodes, force, verbose)
        for s, r in ex.map(compile_one, jobs):
            if r.returncode != 0:
                sys.stderr.write(r.stdout + r.stderr)
                raise RuntimeError("hipcc failed on %s" % s)
            if verbose and r.stderr:
                sys.stderr.write(r.stderr)
        nodes.result()
    if jobs or force or _stale(LIB, objs):
        cmd = [hipcc, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", LIB] + objs + ["-ldl"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
