"""Builds libtmac_cuda.so in-tree: every .cu under csrc/ compiled for sm_100a
(B200) with nvcc, FMA contraction off (-fmad=false) because results must match
the reference's fp32/fp64 roundings bit for bit.  Then, where torch is there to
compile against, _serving.so, the CPython module that takes torch tensors to the
batched decode operators; nothing else needs it."""
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libtmac_cuda.so")
BINDING = os.path.join(HERE, "host", "serving_binding.cpp")
BINDING_OUT = os.path.join(HERE, "_serving.so")
CXX = os.environ.get("CXX", "g++")
NVCC = os.environ.get("NVCC", shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-fmad=false", "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def deps():
    return sources() + sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))) + [
        os.path.join(HERE, "..", "include", "tmac_cuda.h"), os.path.abspath(__file__)]


def up_to_date():
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(d) <= t for d in deps())


def binding_needs():
    """What _serving.so cannot be compiled without and is not here, or None."""
    if importlib.util.find_spec("torch") is None:
        return "torch is not installed"
    import torch
    if torch.version.cuda is None:
        return "torch is built without CUDA"
    if not shutil.which(CXX):
        return f"no C++ compiler ({CXX})"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "no Python headers"
    return None


def built_against():
    """The installations that _serving.so is compiled for."""
    import torch
    return f"torch {torch.__version__} {os.path.dirname(torch.__file__)}, Python {sys.version}\n"


def build_binding(force=False, verbose=False):
    """Compiles _serving.so against the installed torch (host code only)."""
    sources = (BINDING, os.path.join(HERE, "..", "include", "tmac_cuda.h"), os.path.abspath(__file__))
    stamp = os.path.join(HERE, "_build", os.path.basename(BINDING_OUT) + ".for")
    if not force and os.path.exists(BINDING_OUT) and all(os.path.getmtime(s) <= os.path.getmtime(BINDING_OUT) for s in sources) and (
            os.path.exists(stamp) and open(stamp).read() == built_against()):
        return BINDING_OUT
    import torch
    t = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(NVCC))), "include")
    tmp = BINDING_OUT + ".tmp"
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", BINDING, "-o", tmp, f"-I{t}/include", f"-I{t}/include/torch/csrc/api/include",
           f"-I{sysconfig.get_paths()['include']}", f"-I{cuda}", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f"-L{t}/lib", "-lc10", "-ltorch_cpu", "-ltorch_python", "-lc10_cuda", f"-L{HERE}", "-l:libtmac_cuda.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING_OUT)
    os.makedirs(os.path.dirname(stamp), exist_ok=True)
    with open(stamp, "w") as f:
        f.write(built_against())
    return BINDING_OUT


def build(force=False, verbose=False, jobs=8):
    out = build_library(force, verbose, jobs)
    missing = binding_needs()
    if missing:
        print(f"{os.path.basename(BINDING_OUT)} (the batched decode operators on torch tensors) is not built: {missing}", file=sys.stderr)
    else:
        build_binding(force, verbose)
    return out


def build_library(force=False, verbose=False, jobs=8):
    if not force and up_to_date():
        return OUT
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    procs, objs = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        if len([p for p in procs if p[1].poll() is None]) >= jobs:
            procs[0][1].wait()
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if out.strip():
            print(out, file=sys.stderr)
        if p.returncode != 0:
            failed = True
            print(f"nvcc failed on {src}", file=sys.stderr)
    if failed:
        raise RuntimeError("libtmac_cuda.so build failed")
    tmp = OUT + ".tmp"
    cmd = [NVCC, *ARCH, "-shared", "-o", tmp, *objs, "-lcuda"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(OUT)
