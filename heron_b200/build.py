"""Builds libheron_b200.so in-tree with nvcc for sm_100a.

    python -m heron_b200.build [--force] [--verbose]

The library is the package's only compute path.  nvcc cross-compiles without a GPU.  Where torch can be
imported, the C++ front end of some of its operators is built beside it; a host of the C ABI needs neither.
"""
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
TARGET = os.path.join(HERE, "libheron_b200.so")
SOURCES = [os.path.join(CSRC, "hb_api.cu")]
HEADER = os.path.join(HERE, os.pardir, "include", "heron_b200.h")
# the C++ front end of the grouped and 4-bit operators (a CPython extension next to the library)
FRONT = os.path.join(HERE, "_front" + sysconfig.get_config_var("EXT_SUFFIX"))
FRONT_SOURCE = os.path.join(CSRC, "hb_front.cpp")


def deps():
    """Everything the one translation unit includes: all of csrc/ and the public header."""
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))] + [HEADER]


NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC", "-cudart", "static",
]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def is_stale():
    if not os.path.exists(TARGET):
        return True
    t = os.path.getmtime(TARGET)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps())


def _run(cmd, target, verbose):
    """Runs a compiler command with its output beside the target and moved into place, so that a
    reader never sees a half-written file."""
    tmp = target + ".tmp.%d" % os.getpid()
    cmd = cmd + ["-o", tmp]
    if verbose:
        print(" ".join(cmd))
    try:
        subprocess.check_call(cmd)
        os.replace(tmp, target)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)


def cuda_include():
    """The headers of the toolkit that nvcc() belongs to."""
    cc = nvcc()
    return os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(cc) or cc))), "include")


def front_key():
    """What the front end is built for: it links torch's C++ library, which promises no stable interface.  The extension
    carries it as `built_for`, and another one is neither taken for up to date nor called."""
    import torch
    return "heron_b200 front end for torch %s" % torch.__version__


def front_is_stale():
    if not os.path.exists(FRONT):
        return True
    t = os.path.getmtime(FRONT)
    if any(os.path.getmtime(s) > t for s in (FRONT_SOURCE, HEADER, os.path.abspath(__file__))):
        return True
    with open(FRONT, "rb") as f:
        return front_key().encode() + b"\0" not in f.read()


def build_front(force=False, verbose=False):
    """The front end, linked against the library beside it and torch's own libraries."""
    if not force and not front_is_stale():
        return FRONT
    import torch
    from torch.utils import cpp_extension
    inc = cpp_extension.include_paths() + [cuda_include(), sysconfig.get_paths()["include"]]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    _run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
          '-DHB_FRONT_KEY="%s"' % front_key()]
         + [f for i in inc for f in ("-isystem", i)] + [FRONT_SOURCE, "-L" + HERE, "-l:libheron_b200.so", "-L" + lib,
         "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"], FRONT, verbose)
    return FRONT


def build(force=False, verbose=False, extra_flags=()):
    """Builds what is out of date and returns the library's path.  The front end is left out, with a word on stderr, where
    torch, its headers or a C++ compiler are missing: kernels.py does its work without it."""
    build_library(force, verbose, extra_flags)
    try:
        build_front(force, verbose)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        print("heron_b200: front end not built (%s: %s)" % (type(e).__name__, e), file=sys.stderr)
    return TARGET


def build_library(force=False, verbose=False, extra_flags=()):
    """Diagnostic probe modes (knob ``probe``) are compiled in only when HB_PROBES=1 is set in the
    environment; the shipped library has none of their branches."""
    if not force and not is_stale():
        return TARGET
    if os.environ.get("HB_PROBES") == "1":
        extra_flags = list(extra_flags) + ["-DHB_PROBES"]
    _run([nvcc()] + NVCC_FLAGS + list(extra_flags) + SOURCES, TARGET, verbose)
    return TARGET


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True,
          extra_flags=["-Xptxas", "-v"] if "--verbose" in sys.argv else [])
