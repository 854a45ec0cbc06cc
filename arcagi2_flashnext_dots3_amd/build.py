"""Build the gfx950 C-ABI library (libspmla_gfx950.so) in-tree with hipcc.

Every .hip file under csrc/ is compiled to an object (in parallel) and linked into one shared library next to
this file; the Python loader (_lib.py) and the tests load that file. Objects go to _build/ (git-ignored).
csrc/py_call.cpp becomes the extension module _native (the loader's callables; without Python's headers or a C++
compiler it is left out and the loader calls through ctypes), csrc/py_tensors.cpp the extension module _tensors (the
calls around the cache and the query on tensors; without torch's headers it is left out too, and those calls raise).
All HIP code is compiled with packed fp32 instructions disabled (-packed-fp32-ops), see the feature flag below.
"""
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
REPO = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libspmla_gfx950.so")
NATIVE = os.path.join(HERE, "_native" + sysconfig.get_config_var("EXT_SUFFIX"))
TENSORS = os.path.join(HERE, "_tensors" + sysconfig.get_config_var("EXT_SUFFIX"))
CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
FLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", "-Wno-unused-command-line-argument", "-I", CSRC, "-I", os.path.join(REPO, "include")]


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in r.stderr.splitlines() if "packed-fp32-ops" not in l and l.strip())
    if r.returncode != 0:
        raise RuntimeError(f"build failed: {' '.join(cmd)}\n{err}")
    return err


def _build_module(src, out, flags=(), libs=(), headers=()):
    inc = sysconfig.get_paths()["include"]
    headers = [os.path.join(inc, "Python.h"), *headers]
    if not all(os.path.exists(h) for h in headers) or shutil.which(CXX.split()[0]) is None:
        if os.path.exists(out):
            os.remove(out)
        return None
    tmp = out + ".tmp"
    _run([*CXX.split(), "-O2", "-std=c++17", "-shared", "-fPIC", "-I", inc, "-I", os.path.join(REPO, "include"), *flags,
          os.path.join(CSRC, src), "-o", tmp, *libs, "-ldl"])
    os.replace(tmp, out)
    return out


def build_native():
    return _build_module("py_call.cpp", NATIVE)


def build_tensors():
    try:
        import torch
        root, abi = os.path.dirname(torch.__file__), int(torch._C._GLIBCXX_USE_CXX11_ABI)
    except ImportError:
        root, abi = "", 1
    inc, lib = os.path.join(root, "include"), os.path.join(root, "lib")
    return _build_module("py_tensors.cpp", TENSORS,
                         [f"-D_GLIBCXX_USE_CXX11_ABI={abi}", "-I", inc, "-I", os.path.join(inc, "torch", "csrc", "api", "include")],
                         ["-L", lib, "-ltorch_python", "-ltorch_cpu", "-lc10"],
                         [os.path.join(inc, "ATen", "ATen.h"), os.path.join(inc, "torch", "csrc", "autograd", "python_variable.h")])


def build(verbose=False):
    srcs = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    bdir = os.path.join(REPO, "_build")
    os.makedirs(bdir, exist_ok=True)
    objs = [os.path.join(bdir, f[:-4] + ".o") for f in srcs]
    jobs = min(len(srcs), int(os.environ.get("MAX_JOBS", "8")))
    with concurrent.futures.ThreadPoolExecutor(jobs) as ex:
        tensors = ex.submit(build_tensors)
        futs = [ex.submit(_run, [HIPCC, *FLAGS, "-c", os.path.join(CSRC, s), "-o", o]) for s, o in zip(srcs, objs)]
        for s, f in zip(srcs, futs):
            msg = f.result()
            if verbose and msg:
                print(f"[build] {s}: {msg}", flush=True)
    tmp = LIB + ".tmp"
    _run([HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", "-o", tmp, *objs])
    os.replace(tmp, LIB)
    build_native()
    tensors.result()          # the library needs nothing of it: whatever this raises, the library is there
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
