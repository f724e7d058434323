"""Build libcoalibi_sm100.so in-tree with nvcc for sm_100a, and the Python binding of the
serving operators (_serving, C++ over PyTorch's headers) that links it.

    python co-alibi_b200/build.py [--force] [--verbose]

Both land in co-alibi_b200/co_alibi_attn/ next to the Python package that loads
them.  Each is rebuilt only when a source is newer than it.  The library needs nvcc alone;
where PyTorch (with CUDA), Python's headers or a C++ compiler are missing, the binding is
left out with a note, and the serving operators' Python calls say so.
"""
import argparse
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
PKG = os.path.join(HERE, "co_alibi_attn")
OUT = os.path.join(PKG, "libcoalibi_sm100.so")
BINDING_SRC = os.path.join(CSRC, "binding.cpp")
BINDING = os.path.join(PKG, "_serving" + sysconfig.get_config_var("EXT_SUFFIX"))

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr", "--threads", "0",
    "-Xptxas", "-v",
]


def nvcc_path():
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))
                  + glob.glob(os.path.join(INCLUDE, "*.h")))


def needs_build():
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    return any(os.path.getmtime(s) > t for s in sources())


def build(force=False, verbose=False, binding=None):
    """Returns the library's path.  ``binding``: True to fail where it cannot be built."""
    build_library(force, verbose)
    missing = binding_lacks()
    if not missing:
        build_binding(force, verbose)
    elif binding:
        raise RuntimeError(f"the binding of the serving operators needs {missing}")
    else:
        sys.stderr.write(f"build.py: the binding of the serving operators is left out: it needs {missing}\n")
    return OUT


def binding_lacks():
    """What the binding needs and this machine has not, or None."""
    try:
        import torch
    except ImportError as e:
        return f"PyTorch ({e})"
    if not glob.glob(os.path.join(os.path.dirname(torch.__file__), "lib", "*c10_cuda*")):
        return "PyTorch with CUDA"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers (Python.h)"
    if shutil.which(cxx_path()) is None:
        return f"a C++ compiler ({cxx_path()} not found)"
    return None


def cxx_path():
    return os.environ.get("CXX", "g++")


def _run(cmd, verbose, what):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n" + res.stderr[-4000:])
    return res


def build_library(force=False, verbose=False):
    if not force and not needs_build():
        return
    cu = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    tmp = OUT + ".tmp"
    res = _run([nvcc_path(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, *cu, "-o", tmp], verbose, "nvcc")
    os.replace(tmp, OUT)
    with open(OUT + ".ptxas.txt", "w") as f:
        f.write("\n".join(l for l in res.stderr.splitlines() if "ptxas" in l or "registers" in l
                          or "spill" in l or "smem" in l))


def build_binding(force=False, verbose=False):
    header = os.path.join(INCLUDE, "coalibi.h")
    if not force and os.path.exists(BINDING) and all(
            os.path.getmtime(s) <= os.path.getmtime(BINDING) for s in (BINDING_SRC, header)):
        return
    import torch  # for its headers and libraries; nothing of it runs
    home = os.path.dirname(torch.__file__)
    inc = [sysconfig.get_paths()["include"], os.path.join(home, "include"),
           os.path.join(home, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include"), INCLUDE]
    lib = os.path.join(home, "lib")
    tmp = BINDING + ".tmp"
    _run([cxx_path(), "-O2", "-std=c++17", "-fPIC", "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *sum((["-isystem", i] for i in inc), []),
          BINDING_SRC, "-o", tmp, "-L", PKG, "-l:libcoalibi_sm100.so", "-Wl,-rpath,$ORIGIN", "-L", lib,
          f"-Wl,-rpath,{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"],
         verbose, "g++")
    os.replace(tmp, BINDING)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
