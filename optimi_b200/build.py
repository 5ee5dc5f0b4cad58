"""Builds the sm_100a kernel library in-tree, optimi_b200/lib/liboptimi_b200.so, and beside it _host.so, the host side of
optimi_b200/activations.py in C++ (autograd nodes and the calls of the library's C ABI; g++ and torch's headers).  The
library does not depend on torch: each of the two has a stamp of its own, and another torch makes only _host.so stale.

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
HEADER = os.path.join(os.path.dirname(PKG), "include", "optimi_b200.h")
DEPS = [SRC, os.path.join(PKG, "csrc", "mta_common.cuh"), os.path.join(PKG, "csrc", "optimizer_ops.cuh"),
        *ACTIVATION_SRCS, os.path.join(PKG, "csrc", "activation_common.cuh"), os.path.join(PKG, "csrc", "activation_offsets.h"),
        HEADER]  # fmt: skip
HOST_DEPS = [HOST_SRC, HEADER]
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "liboptimi_b200.so")
HOST_LIB = os.path.join(LIB_DIR, "_host.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-fmad=false", "-prec-div=true",
    "-prec-sqrt=true", "-ftz=false", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
]  # fmt: skip

HOST_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=1", "-DTORCH_EXTENSION_NAME=_host"]


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
    return [find_gxx(), *HOST_FLAGS, *[f"-I{d}" for d in include], "-c", "-o", obj, HOST_SRC]


def host_link(obj: str, lib: str, out: str) -> list[str]:
    libs = os.path.join(torch_dir(), "lib")
    return [find_gxx(), "-shared", "-o", out, obj, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            f"-L{os.path.dirname(lib)}", "-l:liboptimi_b200.so", "-Wl,-rpath,$ORIGIN"]  # fmt: skip


STAMP, HOST_STAMP = LIB + ".srchash", HOST_LIB + ".srchash"


def _hash(flags: list[str], files: list[str]) -> str:
    h = hashlib.sha256(" ".join(flags).encode())
    for d in files:
        with open(d, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def source_hash() -> str:
    return _hash(NVCC_FLAGS, DEPS)


def host_source_hash() -> str:
    return _hash(HOST_FLAGS, [*HOST_DEPS, os.path.join(torch_dir(), "version.py")])


def _current(lib: str, stamp: str, wanted) -> bool:
    if not (os.path.exists(lib) and os.path.exists(stamp)):
        return False
    with open(stamp) as fh:
        return fh.read().strip() == wanted()


def up_to_date() -> bool:
    """True when the library was built from the sources as they are now (content hash, not mtime)."""
    return _current(LIB, STAMP, source_hash)


def host_up_to_date() -> bool:
    """The same of _host.so, with the installed torch."""
    return _current(HOST_LIB, HOST_STAMP, host_source_hash)


N_PARTS = 3  # the step source compiles as independent translation units (OPTIMI_PART), built in parallel


def _install(fresh: str, lib: str, stamp: str, wanted: str) -> None:
    if os.path.exists(stamp):
        os.remove(stamp)  # never a current stamp beside an older library
    os.replace(fresh, lib)
    with open(stamp + ".tmp", "w") as fh:
        fh.write(wanted)
    os.replace(stamp + ".tmp", stamp)


def _run(cmd: list[str]) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("link failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)


def build(force: bool = False, verbose: bool = False, library: bool = True, host: bool = True) -> str:
    """Compiles the library and _host.so (`library`, `host`: whether it is asked for) unless they are current.  Safe against
    several processes arriving at once (the ranks of a multi-GPU job importing the package with a stale library): one
    builds under a file lock, into a private directory, and moves the result into place in one step; the others wait
    and find it current."""

    def stale() -> tuple[bool, bool]:
        return library and (force or not up_to_date()), host and (force or not host_up_to_date())

    if not any(stale()):
        return LIB
    import fcntl
    import tempfile

    os.makedirs(LIB_DIR, exist_ok=True)
    with open(os.path.join(LIB_DIR, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        make_library, make_host = stale()  # another process may have built while this one waited
        with tempfile.TemporaryDirectory(dir=LIB_DIR, prefix=".build-") as tmp:
            cmds, objs = [], []
            if make_library:
                nvcc, ccbin = find_nvcc(), ["-ccbin", find_gxx()]
                compile_flags = [f for f in NVCC_FLAGS if f not in ("-shared", "--use-local-env")]
                units = [(SRC, [f"-DOPTIMI_PART={part}"]) for part in range(N_PARTS)] + [(src, []) for src in ACTIVATION_SRCS]
                for number, (src, defines) in enumerate(units):
                    objs.append(os.path.join(tmp, f"part{number}.o"))
                    cmds.append([nvcc, *ccbin, *compile_flags, *(["-Xptxas", "-v"] if verbose else []), *defines, "-c", "-o", objs[-1], src])
            host_obj = os.path.join(tmp, "host.o")
            if make_host:
                cmds.append(host_compile(host_obj))
            procs = [(cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)) for cmd in cmds]
            log = ""
            for cmd, p in procs:
                out, err = p.communicate()
                log += out + err
                if p.returncode != 0:
                    raise RuntimeError("compilation failed:\n" + " ".join(cmd) + "\n" + out + err)
            if make_library:
                fresh = os.path.join(tmp, "liboptimi_b200.so")
                _run([nvcc, *ccbin, "-shared", "-o", fresh, *objs])
                _install(fresh, LIB, STAMP, source_hash())
            if make_host:
                fresh = os.path.join(tmp, "_host.so")
                _run(host_link(host_obj, LIB, fresh))
                _install(fresh, HOST_LIB, HOST_STAMP, host_source_hash())
        if verbose:
            print(log)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
