"""Builds thunderkittens_b200/libtkb200.so from csrc/*.cu with nvcc for sm_100a, and on top of it, for the Python and torch that run
this, the module thunderkittens_b200/_torch_ops.<python's tag>.so from csrc/torch_ops.cpp with the host compiler (in-tree).  Without torch
or a host compiler the C library is all that is built.

    python -m thunderkittens_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU.  Objects go to thunderkittens_b200/_obj/ (git-ignored).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_obj")
LIB = os.path.join(HERE, "libtkb200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops" + sysconfig.get_config_var("EXT_SUFFIX"))
CXX = "g++"
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.path.join(CUDA_HOME, "bin", "nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v"]
# per-file extra flags
EXTRA = {"quantize_fast.cu": ["--use_fast_math"]}


def sources() -> list[str]:
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps() -> list[str]:
    inc = os.path.join(os.path.dirname(HERE), "include")
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cpp")] + [os.path.join(inc, f) for f in os.listdir(inc)] + [__file__]


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJ, src[:-3] + ".o")
    if not force and os.path.exists(obj) and all(os.path.getmtime(d) <= os.path.getmtime(obj) for d in _deps()):
        return obj
    cmd = [NVCC, *ARCH, *COMMON, *EXTRA.get(src, []), "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    log = os.path.join(OBJ, src[:-3] + ".log")
    with open(log, "w") as f:
        f.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"nvcc failed on {src}")
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=8) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose), sources()))
    if force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    _build_torch_ops(force)
    return LIB


def _build_torch_ops(force: bool) -> None:
    """The module of the int8 and norm calls; a module that another torch was built with is replaced."""
    try:
        import torch
    except ImportError:
        torch = None
    if torch is None or shutil.which(CXX) is None:
        print(f"{LIB} is built; {TORCH_OPS}, which ops.int8_* and the norms of ops need, is not: {'no torch' if torch is None else 'no ' + CXX}", file=sys.stderr)
        return
    src = os.path.join(CSRC, "torch_ops.cpp")
    deps = [src, os.path.join(os.path.dirname(HERE), "include", "tkb200.h"), __file__]
    stamp = os.path.join(OBJ, os.path.basename(TORCH_OPS) + ".torch")                 # the torch that it was built with
    try:
        with open(stamp) as f:
            built_with = f.read()
    except OSError:
        built_with = None
    if not force and built_with == torch.__version__ and os.path.exists(TORCH_OPS) and all(os.path.getmtime(d) <= os.path.getmtime(TORCH_OPS) for d in deps):
        return
    torch_dir = os.path.dirname(torch.__file__)
    include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(CUDA_HOME, "include")]
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DTKB_TORCH_VERSION="{torch.__version__}"',
           *(a for d in include for a in ("-isystem", d)), src, "-o", TORCH_OPS, "-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN",
           "-L" + os.path.join(torch_dir, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{CXX} failed on torch_ops.cpp")
    with open(stamp, "w") as f:
        f.write(torch.__version__)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
