"""Builds libssm_b200.so (the C-ABI selective-scan library) in-tree for sm_100a.

    python -m mamba_ssm_benchmark_b200.build            # incremental
    python -m mamba_ssm_benchmark_b200.build --force    # rebuild everything

Each .cu file under csrc/ is compiled by nvcc in parallel into _build/, then linked into
mamba_ssm_benchmark_b200/_C/libssm_b200.so with the CUDA runtime linked statically, so the
library needs only the driver at run time.  nvcc cross-compiles: no GPU is needed to build.
csrc/torch_glue.cpp (torch tensors and autograd over that library) becomes _C/_glue.so, compiled
by the host compiler against the installed torch at the same time.
"""

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
OUT_DIR = os.path.join(PKG, "_C")
LIB = os.path.join(OUT_DIR, "libssm_b200.so")
GLUE_SRC = os.path.join(CSRC, "torch_glue.cpp")
GLUE = os.path.join(OUT_DIR, "_glue.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC]


def nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _compile(src, obj, verbose):
    cmd = [nvcc()] + ARCH + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stderr[-8000:]}")
    return r.stderr


def _compile_glue(obj):
    """torch_glue.cpp against the installed torch (headers only; linked by _link_glue)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    paths = [INCLUDE, sysconfig.get_paths()["include"], cuda] + include_paths()
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_glue",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += [f for path in paths for f in ("-isystem", path)] + ["-c", GLUE_SRC, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"the host compiler failed for torch_glue.cpp:\n{r.stderr[-8000:]}")
    return r.stderr


def _link_glue(obj):
    import torch
    tmp = GLUE + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", tmp, obj, "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-L" + OUT_DIR, "-l:" + os.path.basename(LIB),
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-8000:]}")
    os.replace(tmp, GLUE)


def build(force=False, verbose=False, jobs=None):
    """Compiles every CUDA source for sm_100a and the torch glue, and links both libraries; returns the path of
    libssm_b200.so."""
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(OUT_DIR, exist_ok=True)
    newest_header = max(os.path.getmtime(h) for h in _headers())
    todo, objs = [], []
    for src in _sources():
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header):
            todo.append((src, obj))
    glue_obj = os.path.join(BUILD, "torch_glue.o")
    glue = force or not os.path.exists(glue_obj) or os.path.getmtime(glue_obj) < max(os.path.getmtime(GLUE_SRC),
                                                                                     newest_header)
    if todo or glue:
        jobs = jobs or min(len(todo) + 1, os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(jobs) as ex:
            futs = {ex.submit(_compile, s, o, verbose): s for s, o in todo}
            if glue:
                futs[ex.submit(_compile_glue, glue_obj)] = GLUE_SRC
            for f in cf.as_completed(futs):
                log = f.result()
                if verbose and log:
                    sys.stderr.write(log)
    if todo or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc()] + ARCH + ["-shared", "-Xcompiler", "-fPIC", "-cudart", "static", "-o", tmp] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr[-8000:]}")
        os.replace(tmp, LIB)
    if glue or not os.path.exists(GLUE) or os.path.getmtime(GLUE) < os.path.getmtime(glue_obj):
        _link_glue(glue_obj)
    return LIB


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="pass -Xptxas -v and print its report")
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args(argv)
    print(build(force=args.force, verbose=args.verbose, jobs=args.jobs))


if __name__ == "__main__":
    main()
