"""Builds libo1b200.so (the CUDA kernels + C ABI) in-tree with nvcc for sm_100a, and _binding.so (the Python calls
whose host time counts, on torch tensors) with g++ where there is a torch with CUDA: the library itself needs none.

Run as a script or call build(); nothing is JIT-compiled at import time, so
the built library travels with the source tree.
"""
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libo1b200.so")
SOURCES = ["gemm_tc.cu", "attn_tc.cu", "elementwise.cu", "vision.cu", "sched.cu", "lora.cu", "lora_static.cu", "kvcache.cu", "pages.cu", "rotary.cu", "decode.cu", "sp.cu", "host.cu", "weights.cu", "engine.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


BINDING, BINDING_SRC = os.path.join(HERE, "_binding.so"), os.path.join(CSRC, "binding.cpp")


def _binding():
    """(object file, which names the torch it is for; commands that compile and link) of the native module, or (None, why there is none)."""
    import sysconfig
    try:
        import torch
    except ImportError:
        return None, "there is no torch"
    root = os.path.dirname(torch.__file__)
    if not os.path.exists(os.path.join(root, "lib", "libtorch_cuda.so")):
        return None, f"torch {torch.__version__} is without CUDA"
    obj = os.path.join(CSRC, f"binding.{torch.__version__}.o")
    compile_ = (["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
                + [f"-I{d}" for d in (sysconfig.get_paths()["include"], os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                                      os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include"))]
                + ["-c", BINDING_SRC, "-o", obj])
    link = ["g++", "-shared", obj, "-o", BINDING, f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10_cuda", "-lc10"]
    return obj, (compile_, link)


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose=False, force=False):
    """O1_NVCC_EXTRA (environment): extra nvcc flags, e.g. -DO1_ATTN_P_F16=0; changing it needs force."""
    nvcc = _nvcc()
    extra = os.environ.get("O1_NVCC_EXTRA", "").split()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(HERE, "..", "include", "o1_b200.h"))
    objs = []
    procs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(CSRC, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = [nvcc] + NVCC_FLAGS + extra + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    binding, how = _binding()
    if binding is None:
        sys.stderr.write(f"{os.path.basename(BINDING)} is not built ({how}): KvCache, KvPages, Rotary, Decoder and residual_norm are not to be had from Python\n")
    elif force or _stale(binding, [BINDING_SRC, headers[-1]]):
        for old in glob.glob(os.path.join(CSRC, "binding.*.o")):       # of another torch
            os.remove(old)
        procs.append(("binding.cpp", subprocess.Popen(how[0], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed = True
            sys.stderr.write(f"--- {src} failed\n{out}\n")
        elif verbose:
            sys.stderr.write(f"--- {src}\n{out}\n")
    if failed:
        raise RuntimeError("nvcc compilation failed")
    if force or procs or _stale(LIB, objs):
        cmd = [nvcc, "-shared", "-o", LIB] + objs + ["-Xlinker", "-Bsymbolic", "-lcudart"]
        subprocess.run(cmd, check=True)
    if binding is not None and (force or _stale(BINDING, [binding])):
        subprocess.run(how[1], check=True)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
