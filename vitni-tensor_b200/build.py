"""Build the sm_100a shared library ``vtq/libvtq.so`` in-tree with nvcc, and, where torch and its
headers are there, the torch binding of the batched serving operators, ``vtq/_serving.so``, with the
host compiler (``vtq.serving`` says so where it is missing; the C library does not need it).

Usage: python vitni-tensor_b200/build.py [--force]
Every .cu under csrc/ is compiled for sm_100a only, with fp32 contraction
disabled (-fmad=false): bit parity with the reference depends on every fp32
multiply and add being rounded separately.
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "vtq", "libvtq.so")
BINDING = os.path.join(HERE, "vtq", "_serving.so")
OBJ = os.path.join(HERE, "_build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true",
    "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
    "-Xptxas", "-warn-spills",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def deps():
    out = []
    for d in (CSRC, os.path.join(HERE, "..", "include")):
        out += [os.path.join(d, f) for f in os.listdir(d) if not f.endswith(".cpp")]
    return out


def build(force=False, verbose=False):
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJ, exist_ok=True)
    newest_dep = max(os.path.getmtime(p) for p in deps())
    objs = []
    for src in sources():
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep:
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    if force or not os.path.exists(OUT) or any(os.path.getmtime(o) > os.path.getmtime(OUT) for o in objs):
        cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", OUT, *objs]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return OUT


def build_binding(force=False, verbose=False):
    """vtq/_serving.so from csrc/serving_bind.cpp, against this interpreter's torch and libvtq.so."""
    src, out = os.path.join(CSRC, "serving_bind.cpp"), BINDING
    header = os.path.join(HERE, "..", "include", "vtq.h")
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(p) for p in (src, header)):
        return out
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    nvcc = shutil.which(os.environ.get("NVCC", "nvcc"))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc)))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", src, "-o", out,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"),
           *("-I" + p for p in cpp_extension.include_paths()), "-L" + lib, "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-ltorch_cuda", "-lc10", "-lc10_cuda", "-L" + os.path.join(HERE, "vtq"), "-l:libvtq.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return out


def main(args):
    force = "--force" in args
    lib = build(force=force, verbose=True)
    try:
        out = [lib, build_binding(force=force, verbose=True)]
    except (ImportError, OSError, TypeError, subprocess.CalledProcessError) as e:
        if os.path.exists(BINDING):
            os.remove(BINDING)  # of an earlier build: it may not fit this library
        print(f"{BINDING} is not built ({e}): vtq.serving needs torch, its headers and a host compiler", file=sys.stderr)
        out = [lib]
    print(*out, sep="\n")
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
