"""Ahead-of-time build of the native library (sm_100a only, in-tree).

`python -m yirage_b200.build` compiles every csrc/*.cu into yirage_b200/libypk.so with nvcc:
the host side of the C ABI (ypk_abi.cu) and one translation unit per kernel variant
(megakernel_decode.cu, megakernel_decode_tp.cu, megakernel_wide.cu, megakernel_moe.cu), each
of which includes the task runners (runners.cuh) and so owns its copies of them, and the
handle-free operators (op_*.cu); relocatable device code linked at the end.  Then g++ compiles
the Python binding of the serving operators' hot calls (serving_binding.cpp) into
yirage_b200/_serving.so, which needs torch's headers and libypk.so.  There is no per-model JIT: shapes travel in the task table at
run time, unlike the reference which runs nvcc for every graph
(python/yirage/persistent_kernel.py:1138-1318).
"""
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libypk.so")
BINDING = os.path.join(HERE, "_serving.so")
BINDING_SOURCE = os.path.join(CSRC, "serving_binding.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-rdc=true", "--threads", "0",
    # every runner is called from a kernel of 288 threads (one CTA per SM): 168 registers per
    # thread is what such a kernel can have, and a callee may not use more than its caller
    "-maxrregcount", "168",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-v",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = deps + [os.path.join(HERE, "..", "include", "ypk.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _run(cmd, verbose, what):
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed")


def _binding_command():
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    libs = os.path.join(base, "lib")
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", BINDING, BINDING_SOURCE,
            f"-I{os.path.join(base, 'include')}", f"-I{sysconfig.get_paths()['include']}",
            f"-I{os.path.join(cuda, 'include')}", f"-L{HERE}", "-l:libypk.so", f"-L{libs}", "-ltorch_python",
            "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"]


def _binding_lacks():
    """What the Python binding needs and this machine has not, or None."""
    if shutil.which("g++") is None:
        return "g++"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    try:
        import torch
    except ImportError:
        return "torch"
    if not os.path.isdir(os.path.join(os.path.dirname(torch.__file__), "include", "torch")):
        return "torch's headers"
    return None


def build(force=False, verbose=False):
    """Compile libypk.so and _serving.so where missing or older than their sources.  libypk.so, all
    that a C host needs, takes nvcc alone; where what the Python binding takes is missing, that is
    left out with a message and serving.py raises when it is used."""
    native = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cpp")]
    if force or _stale(LIB, native):
        nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
        if not os.path.exists(nvcc):
            raise RuntimeError("nvcc not found; the native library cannot be built")
        _run([nvcc] + NVCC_FLAGS + ["-o", LIB] + sources() + ["-lcudart"], verbose, "nvcc building libypk.so")
    if force or _stale(BINDING, [BINDING_SOURCE, os.path.join(CSRC, "strided_rows.h")]):
        lacking = _binding_lacks()
        if lacking is None:
            _run(_binding_command(), verbose, "g++ building _serving.so")
        else:
            if os.path.exists(BINDING):      # of other sources: its structures may not be today's
                os.remove(BINDING)
            sys.stderr.write(f"_serving.so, the Python binding of the serving operators, is not built: no {lacking}\n")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
