"""Builds libenvgemm.so in-tree for sm_100a (nvcc cross-compiles; no GPU needed)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = [os.path.join(HERE, "csrc", "envgemm.cu")]
INCLUDE = os.path.join(os.path.dirname(HERE), "include")


def deps():
    """Every source and header the library is compiled from."""
    csrc = os.path.join(HERE, "csrc")
    files = [os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith((".cu", ".cuh", ".hpp", ".h"))]
    return files + [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith((".h", ".hpp"))]
OUT = os.path.join(HERE, "lib", "libenvgemm.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC,-O3", "-shared"]


# The torch side of the Python binding (operand checks in one step); the library itself needs no torch,
# and the binding goes on without this extension.
VIEWS_SRC = os.path.join(HERE, "csrc", "views.cpp")
VIEWS = os.path.join(HERE, "lib", "_views.so")


def views_stamp():
    """What lib/_views.so has to be built from and for: its source, this torch and this interpreter."""
    import hashlib
    import sysconfig

    import torch

    with open(VIEWS_SRC, "rb") as f:
        src = hashlib.sha256(f.read()).hexdigest()[:16]
    return f"{src} torch {torch.__version__} {sysconfig.get_config_var('SOABI')}"


def build_views(force=False, verbose=True):
    """Builds lib/_views.so against the torch of this interpreter.  Where that cannot be done (no torch, one
    without CUDA, no compiler) there is none afterwards: a warning, and None."""
    try:
        stamp = views_stamp()
        if not force and os.path.exists(VIEWS):
            with open(VIEWS, "rb") as f:
                if stamp.encode() in f.read():
                    return VIEWS
        if os.path.exists(VIEWS):
            os.remove(VIEWS)
        import sysconfig

        import torch
        from torch.utils.cpp_extension import include_paths

        lib = os.path.join(os.path.dirname(torch.__file__), "lib")
        cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               f'-DENVG_VIEWS_STAMP="{stamp}"',
               "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
        cmd += ["-I" + p for p in include_paths()]
        cmd += [VIEWS_SRC, "-L" + lib, "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-o", VIEWS]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    except (ImportError, OSError, AttributeError, subprocess.CalledProcessError) as e:
        if os.path.exists(VIEWS):
            os.remove(VIEWS)
        print(f"warning: lib/_views.so was not built, calls on CUDA tensors take about 5 us longer ({e})", file=sys.stderr, flush=True)
        return None
    return VIEWS


def needs_build():
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    return any(os.path.getmtime(p) > t for p in deps())


def build(force=False, verbose=True):
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    if force or needs_build():
        cmd = [NVCC] + FLAGS + SRC + ["-o", OUT]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    build_views(force, verbose)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
