"""Builds the sm_100a kernel library in-tree, optimi_b200/lib/liboptimi_b200.so, and beside it _host.so, the host side of
optimi_b200/activations.py in C++ (autograd nodes and the calls of the library's C ABI; g++ and torch's headers).

    python -m optimi_b200.build [--force]

nvcc cross-compiles without a GPU.  Flags that matter for parity: -fmad=false (the kernels fuse
multiply-adds only where they say so with __fmaf_rn), default IEEE division and square root.
"""

from __future__ import annotations

import hashlib
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(PKG, "csrc", "optimi_b200.cu")
ACTIVATION_SRCS = [os.path.join(PKG, "csrc", "activation_ops.cu"), os.path.join(PKG, "csrc", "weight_gradient.cu")]
HOST_SRC = os.path.join(PKG, "csrc", "activations_host.cpp")
DEPS = [SRC, HOST_SRC, os.path.join(PKG, "csrc", "mta_common.cuh"), os.path.join(PKG, "csrc", "optimizer_ops.cuh"),
        *ACTIVATION_SRCS, os.path.join(PKG, "csrc", "activation_common.cuh"), os.path.join(PKG, "csrc", "activation_offsets.h"),
        os.path.join(os.path.dirname(PKG), "include", "optimi_b200.h")]  # fmt: skip
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "liboptimi_b200.so")
HOST_LIB = os.path.join(LIB_DIR, "_host.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-fmad=false", "-prec-div=true",
    "-prec-sqrt=true", "-ftz=false", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
]  # fmt: skip


def find_gxx() -> str:
    """The system's compiler (the environment's CC and CXX may point at a wrapper)."""
    return "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"


def find_nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or add it to PATH)")


def torch_dir() -> str:
    """Where torch is installed (found without importing it)."""
    return next(iter(importlib.util.find_spec("torch").submodule_search_locations))


def host_compile(obj: str) -> list[str]:
    torch, cuda = torch_dir(), os.path.dirname(os.path.dirname(os.path.realpath(find_nvcc())))
    include = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]  # fmt: skip
    return [find_gxx(), "-O2", "-std=c++17", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=1", "-DTORCH_EXTENSION_NAME=_host", *[f"-I{d}" for d in include],
            "-c", "-o", obj, HOST_SRC]  # fmt: skip


def host_link(obj: str, lib: str, out: str) -> list[str]:
    libs = os.path.join(torch_dir(), "lib")
    return [find_gxx(), "-shared", "-o", out, obj, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            f"-L{os.path.dirname(lib)}", "-l:liboptimi_b200.so", "-Wl,-rpath,$ORIGIN"]  # fmt: skip


STAMP = LIB + ".srchash"


def source_hash() -> str:
    h = hashlib.sha256(" ".join(NVCC_FLAGS).encode())
    for d in [*DEPS, os.path.join(torch_dir(), "version.py")]:
        with open(d, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def up_to_date() -> bool:
    """True when the library was built from the sources as they are now (content hash, not mtime)."""
    if not (os.path.exists(LIB) and os.path.exists(HOST_LIB) and os.path.exists(STAMP)):
        return False
    with open(STAMP) as fh:
        return fh.read().strip() == source_hash()


N_PARTS = 3  # the step source compiles as independent translation units (OPTIMI_PART), built in parallel


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library unless it is current.  Safe against several processes arriving at once (the ranks of
    a multi-GPU job importing the package with a stale library): one builds under a file lock, into a private
    directory, and moves the result into place in one step; the others wait and find it current."""
    if not force and up_to_date():
        return LIB
    import fcntl
    import tempfile

    os.makedirs(LIB_DIR, exist_ok=True)
    with open(os.path.join(LIB_DIR, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        if not force and up_to_date():  # another process built it while this one waited
            return LIB
        nvcc = find_nvcc()
        ccbin = ["-ccbin", find_gxx()]
        compile_flags = [f for f in NVCC_FLAGS if f not in ("-shared", "--use-local-env")]
        with tempfile.TemporaryDirectory(dir=LIB_DIR, prefix=".build-") as tmp:
            objs, procs = [], []
            units = [(SRC, [f"-DOPTIMI_PART={part}"]) for part in range(N_PARTS)] + [(src, []) for src in ACTIVATION_SRCS]
            for number, (src, defines) in enumerate(units):
                obj = os.path.join(tmp, f"part{number}.o")
                objs.append(obj)
                cmd = [nvcc, *ccbin, *compile_flags, *(["-Xptxas", "-v"] if verbose else []), *defines, "-c", "-o", obj, src]
                procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
            host_obj = os.path.join(tmp, "host.o")
            cmd = host_compile(host_obj)
            procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
            log = ""
            for cmd, p in procs:
                out, err = p.communicate()
                log += out + err
                if p.returncode != 0:
                    raise RuntimeError("compilation failed:\n" + " ".join(cmd) + "\n" + out + err)
            fresh = os.path.join(tmp, "liboptimi_b200.so")
            fresh_host = os.path.join(tmp, "_host.so")
            for link in ([nvcc, *ccbin, "-shared", "-o", fresh, *objs], host_link(host_obj, fresh, fresh_host)):
                res = subprocess.run(link, capture_output=True, text=True)
                if res.returncode != 0:
                    raise RuntimeError("link failed:\n" + " ".join(link) + "\n" + res.stdout + res.stderr)
            if os.path.exists(STAMP):
                os.remove(STAMP)  # never a current stamp beside an older library
            os.replace(fresh, LIB)
            os.replace(fresh_host, HOST_LIB)
        if verbose:
            print(log)
        with open(STAMP + ".tmp", "w") as fh:
            fh.write(source_hash())
        os.replace(STAMP + ".tmp", STAMP)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
