"""Builds need_b200/_lib/libneed_scan.so from need_b200/csrc with nvcc for sm_100a,
and over it, with the host compiler against torch's headers, need_b200/_lib/_train.so
(the autograd nodes of need_b200.train) and _lm.so (the operators of need_b200.lm).

    python -m need_b200.build            # build if sources changed
    python -m need_b200.build --force

The library is built in-tree so it travels with the repository; there is no
JIT path.  Flags: -gencode arch=compute_100a,code=sm_100a (B200 only), -O3,
-lineinfo (source-level ncu attribution), static cudart.  libneed_scan.so does
not depend on torch.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIBDIR = os.path.join(HERE, "_lib")
LIB = os.path.join(LIBDIR, "libneed_scan.so")
EXT = os.path.join(LIBDIR, "_train.so")
EXT_SOURCE = "train_autograd.cpp"
EXTS = {EXT: EXT_SOURCE, os.path.join(LIBDIR, "_lm.so"): "lm_autograd.cpp"}
EXT_HEADERS = ["torch_common.h"]
SOURCES = ["need_scan.cu", "decode.cu", "sp.cu", "noalloc.cu", "segments.cu", "prologue.cu", "epilogue.cu", "assoc.cu",
           "train_scan.cu", "train_conv.cu", "train_norm.cu", "linear_attention.cu", "linear_attention_umma.cu",
           "linear_attention_step.cu",
           "residual_norm.cu", "token_log_probs.cu"]
HEADERS = ["ptx.cuh", "scan_kernel.cuh", "host_common.h", "umma.cuh", "train_common.cuh", "linear_attention.cuh"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def _older(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _stale() -> bool:
    return _older(LIB, [os.path.join(CSRC, f) for f in SOURCES + HEADERS] + [os.path.join(INCLUDE, "need_scan.h")])


def _ext_stale(ext: str = EXT) -> bool:
    return _older(ext, [os.path.join(CSRC, f) for f in [EXTS[ext]] + EXT_HEADERS] + [os.path.join(INCLUDE, "need_scan.h")])


def _ext_command(ext: str = EXT) -> list:
    """The host compile of a module over torch (no torch import: its headers are found by path).

    The C++ library is named as the shared one that torch runs on: a compiler that finds only
    the archive (a $CXX of its own tree) would link a second copy into the module, whose
    locale is not the one torch's exports have set up, and a stream that formats a number
    there ends the process."""
    import importlib.util
    import sysconfig
    torch_dir = os.path.dirname(importlib.util.find_spec("torch").origin)
    inc = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_path("include"), os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
            f"-DTORCH_EXTENSION_NAME={os.path.basename(ext)[:-3]}", "-DTORCH_API_INCLUDE_EXTENSION_H", f"-I{INCLUDE}",
            *[x for d in inc for x in ("-isystem", d)], os.path.join(CSRC, EXTS[ext]), "-o", ext + ".tmp",
            "-L" + os.path.join(torch_dir, "lib"), "-L" + LIBDIR, "-l:libneed_scan.so", "-lc10", "-lc10_cuda", "-ltorch",
            "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-nostdlib++", "-l:libstdc++.so.6", "-lm", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the shared library and the modules over torch if needed; returns the library's path."""
    os.makedirs(LIBDIR, exist_ok=True)
    if force or _stale():
        _build_lib(verbose)
    procs = []
    for ext, src in EXTS.items():
        if force or _ext_stale(ext):
            cmd = _ext_command(ext)
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            procs.append((ext, src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = []
    for ext, src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"--- {src}\n{out.decode(errors='replace')}")
        else:
            os.replace(ext + ".tmp", ext)
    if failed:
        raise RuntimeError("\n".join(failed))
    return LIB


def _build_lib(verbose: bool) -> None:
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    common = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
              f"-I{INCLUDE}", f"-I{CSRC}", "--expt-relaxed-constexpr"]
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        cmd = common + ["-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"--- {src}\n{out.decode(errors='replace')}")
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-cudart", "static",
           "-Xlinker", "--exclude-libs,ALL"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
