"""Builds the sampler's CUDA library in-tree for sm_100a.

Produces qwen600_engine_b200/libqwen600_sampler.so from csrc/*.cu with nvcc
(no GPU needed: nvcc cross-compiles), and _torch.so, the torch binding of the
scoring, loss and 4-bit lm_head calls, from csrc/qs_torch.cpp.  --fmad=false keeps every fp32
multiply and add separately rounded, as the reference host sampler computes
them; -lineinfo keeps profiler source correlation.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libqwen600_sampler.so")
SOURCES = ["qs_row.cu", "qs_row_wide.cu", "qs_ties.cu", "qs_sort.cu", "qs_api.cu", "qs_static.cu", "qs_lmhead.cu",
           "qs_losses.cu", "qs_w4.cu", "qs_top.cu", "qs_distill.cu", "qs_reorder.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "--fmad=false", "-std=c++17", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
         "-I", OUT_DIR]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def exp_table(verbose: bool = False) -> str:
    """Generates _build/qs_exp_table.inc: the inputs where the host libm's
    expf (what the reference sampler calls) rounds differently from
    qs_exp_rn.  Takes about a minute; redone only when its sources change."""
    os.makedirs(OUT_DIR, exist_ok=True)
    inc = os.path.join(OUT_DIR, "qs_exp_table.inc")
    gen_src = os.path.join(CSRC, "qs_exp_table.c")
    deps = [gen_src, os.path.join(CSRC, "qs_exp.h")]
    if not _stale(inc, deps):
        return inc
    exe = os.path.join(OUT_DIR, "qs_exp_table")
    cc = shutil.which("gcc") or "cc"
    flags = ["-O2", "-ffp-contract=off"]
    try:
        if " fma " in open("/proc/cpuinfo").read():
            flags.append("-mfma")  # hardware fma: same IEEE result, faster scan
    except OSError:
        pass
    r = subprocess.run([cc] + flags + ["-I", CSRC, "-o", exe, gen_src, "-lm"],
                       capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compiling qs_exp_table.c failed:\n{r.stderr}")
    tmp = inc + ".tmp"
    r = subprocess.run([exe, tmp], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"qs_exp_table failed:\n{r.stderr}")
    os.replace(tmp, inc)
    if verbose:
        print(r.stdout.strip())
    return inc


def build(verbose: bool = False, ptxas_info: bool = False, force: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    table = exp_table(verbose)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(table)
    headers.append(os.path.join(ROOT, "include", "qwen600_sampler.h"))
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OUT_DIR, src.replace(".cu", ".o"))
        objs.append(o)
        if force or ptxas_info or _stale(o, [s, __file__] + headers):
            cmd = [nvcc()] + ARCH + FLAGS + ["-c", s, "-o", o]
            if ptxas_info:
                cmd += ["-Xptxas", "-v"]
            if verbose:
                print(" ".join(cmd))
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
            if ptxas_info or verbose:
                sys.stderr.write(r.stderr)
    if force or _stale(LIB, objs):
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    build_binding(verbose, force)
    build_integration(verbose, force)
    return LIB


BINDING = os.path.join(HERE, "_torch.so")
BINDING_MADE_FOR = os.path.join(OUT_DIR, "torch_binding_made_for")  # the torch and Python of the binding there is


def build_binding(verbose: bool = False, force: bool = False) -> str:
    """_torch.so: the scoring, loss and 4-bit lm_head calls for torch tensors
    (csrc/qs_torch.cpp), linked to the sampler library and torch's own; made
    anew for another torch or Python, whose ABI it would not fit."""
    src = os.path.join(CSRC, "qs_torch.cpp")
    deps = [src, os.path.join(ROOT, "include", "qwen600_sampler.h"), __file__]
    import importlib.metadata
    import sysconfig
    made_for = f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"
    try:
        with open(BINDING_MADE_FOR) as f:
            same = f.read() == made_for
    except OSError:
        same = False
    if not force and same and not _stale(BINDING, deps):
        return BINDING

    import torch
    top = os.path.dirname(torch.__file__)
    inc = [os.path.join(ROOT, "include"), os.path.join(top, "include"),
           os.path.join(top, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in inc:
        cmd += ["-isystem" if d.startswith(top) else "-I", d]
    cmd += [src, "-o", BINDING, "-L", HERE, "-lqwen600_sampler", "-Wl,-rpath,$ORIGIN", "-L", os.path.join(top, "lib"),
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building the torch binding failed:\n{r.stderr}")
    with open(BINDING_MADE_FOR, "w") as f:
        f.write(made_for)
    return BINDING


INTEG = os.path.join(ROOT, "integration")
DEMO_LIB = os.path.join(INTEG, "libqs_decode_demo.so")


def build_integration(verbose: bool = False, force: bool = False) -> str:
    """integration/libqs_decode_demo.so: a decode loop written against the
    reference sampler's interface (integration/qs_sampler_compat.h), linked to
    the sampler library."""
    src = os.path.join(INTEG, "decode_demo.cu")
    deps = [src, os.path.join(INTEG, "qs_sampler_compat.h"), os.path.join(ROOT, "include", "qwen600_sampler.h"),
            LIB, __file__]
    if not force and not _stale(DEMO_LIB, deps):
        return DEMO_LIB
    cmd = [nvcc()] + ARCH + ["-O2", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
                             "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include"), "-I", INTEG,
                             src, "-o", DEMO_LIB, "-L", HERE, "-lqwen600_sampler",
                             "-Xlinker", "-rpath,$ORIGIN/../qwen600_engine_b200"]
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building the decode demo failed:\n{r.stderr}")
    return DEMO_LIB


if __name__ == "__main__":
    build(verbose=True, ptxas_info="-v" in sys.argv, force="-f" in sys.argv)
    print(LIB)
