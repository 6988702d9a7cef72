"""Build libsoraku_b200.so (sm_100a) in-tree with nvcc, and the extension module _bind with g++.

Each .cu under csrc/ compiles to an object in _build/ (in parallel), then
nvcc links the shared library next to this file.  Objects are rebuilt when
their source or any header changed.  _bind (csrc/bind.cpp) is the short way from
Python to some of the library's functions.  It is compiled against torch's headers and
this interpreter's: its file name carries the interpreter's ABI, it says which torch it
was compiled against (bind_key), and it is rebuilt when its command or either
changes.  The library does without it (_lib.bind), so that it is no error where it
cannot be built.
"""

from __future__ import annotations

import glob
import os
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libsoraku_b200.so")
BIND = os.path.join(HERE, "_bind" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
BIND_STAMP = os.path.join(BUILD, "bind.txt")  # how BIND was built
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", INCLUDE]


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, hdr_mtime: float, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_mtime):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        sys.stderr.write(res.stderr)
    return obj


def bind_key() -> str:
    """What _bind has to have been compiled against: its headers' inline accessors know how this torch lays out a tensor."""
    import torch

    return f"torch {torch.__version__} {torch.version.git_version} c++11 abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def _build_bind(force: bool) -> None:
    import torch

    src = os.path.join(CSRC, "bind.cpp")
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(NVCC)))
    system = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
              os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DSKB_BIND_KEY="{bind_key()}"', "-I", INCLUDE, *(f"-isystem{p}" for p in system), src, "-o", BIND, "-L",
           os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    stamp = "\n".join(cmd)
    newest = max(os.path.getmtime(p) for p in (src, os.path.join(INCLUDE, "soraku_b200.h")))
    if not force and os.path.exists(BIND) and os.path.getmtime(BIND) >= newest and os.path.exists(BIND_STAMP):
        with open(BIND_STAMP) as f:
            if f.read() == stamp:
                return
    for old in (BIND, BIND_STAMP, os.path.join(HERE, "_bind.so")):  # the last: a name without an ABI, which any interpreter loads
        if os.path.exists(old):
            os.remove(old)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {src}:\n{res.stdout}\n{res.stderr}")
    with open(BIND_STAMP, "w") as f:
        f.write(stamp)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr = _headers_mtime()
    if force:
        for o in glob.glob(os.path.join(BUILD, "*.o")):
            os.remove(o)
    with ThreadPoolExecutor(max_workers=max(1, min(len(srcs) + 1, os.cpu_count() or 4))) as ex:
        bind = ex.submit(_build_bind, force)
        objs = list(ex.map(lambda s: _compile(s, hdr, verbose), srcs))
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc link failed:\n{res.stdout}\n{res.stderr}")
    try:
        bind.result()
    except Exception as e:  # no torch, no headers, no g++: the library stands
        warnings.warn(f"{os.path.basename(BIND)} was not built, calls go the longer way through ctypes: {e}", RuntimeWarning,
                      stacklevel=2)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
