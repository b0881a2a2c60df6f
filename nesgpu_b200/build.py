"""Builds ``nesgpu_b200/lib/libnesgpu_b200.so`` (sm_100a only) from ``nesgpu_b200/csrc/*.cu`` and the extension module
``nesgpu_b200/_host.so`` (host code that allocates through PyTorch and calls the library) from ``csrc/*_host.cpp``.

Usage: ``python -m nesgpu_b200.build [--force] [--verbose]``.  nvcc cross-compiles without a
GPU; the shared library is kept in-tree next to the package.  What is newer than its sources is left as it is, the extension
module only if it was also built for this PyTorch and this Python.
"""
import concurrent.futures
import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libnesgpu_b200.so")
HOST_PATH = os.path.join(PKG, "_host.so")
OBJ_DIR = os.path.join(PKG, "build")
HOST_TAG = os.path.join(OBJ_DIR, "microscaling_host.tag")      # what the extension module was built for
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def _nvcc():
    return os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps_mtime():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(INCLUDE, "nesgpu_b200.h")]
    return max(os.path.getmtime(f) for f in files)


def _compile(src, verbose):
    obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
    extra = os.environ.get("NES_NVCC_EXTRA", "").split()      # e.g. -DNAME for an instrumented build
    cmd = [_nvcc()] + NVCC_FLAGS + extra + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed for %s:\n%s\n%s" % (src, res.stdout, res.stderr))
    return obj, res.stderr


def _torch_dir():
    import torch
    return os.path.dirname(torch.__file__)


def _compile_host():
    """Object of the extension module: PyTorch's headers, no CUDA code."""
    src, obj = os.path.join(CSRC, "microscaling_host.cpp"), os.path.join(OBJ_DIR, "microscaling_host.o")
    torch_include = os.path.join(_torch_dir(), "include")
    include = [torch_include, os.path.join(torch_include, "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-c", src, "-o", obj] + ["-I" + d for d in include]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed for %s:\n%s\n%s" % (src, res.stdout, res.stderr))
    return obj


def _link_host(obj):
    cmd = ["g++", "-shared", "-o", HOST_PATH, obj, "-L" + LIB_DIR, "-lnesgpu_b200", "-Wl,-rpath,$ORIGIN/lib",
           "-L" + os.path.join(_torch_dir(), "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
           "-lc10_cuda", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("link failed:\n%s\n%s" % (res.stdout, res.stderr))


def _link_library(objs):
    cmd = [_nvcc(), "-shared", "-o", LIB_PATH] + objs + ["-gencode", "arch=compute_100a,code=sm_100a"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("link failed:\n%s\n%s" % (res.stdout, res.stderr))


def _wanted_tag():
    import torch
    return "torch %s, python %s" % (torch.__version__, sysconfig.get_config_var("SOABI"))


def _built_tag():
    try:
        with open(HOST_TAG) as f:
            return f.read()
    except OSError:
        return None


def _is_current(path):
    return os.path.exists(path) and os.path.getmtime(path) >= _deps_mtime()


def build(force=False, verbose=False):
    """Compile every CUDA source for sm_100a and link the shared library, then the extension module.  Returns the
    library's path."""
    os.makedirs(LIB_DIR, exist_ok=True)
    os.makedirs(OBJ_DIR, exist_ok=True)
    library = force or not _is_current(LIB_PATH)
    host = library or not _is_current(HOST_PATH) or _built_tag() != _wanted_tag()
    srcs = sources() if library else []
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as pool:
        host_obj = pool.submit(_compile_host) if host else None
        results = list(pool.map(lambda s: _compile(s, verbose), srcs))
    if verbose:
        for _, log in results:
            sys.stderr.write(log)
    if library:
        _link_library([o for o, _ in results])
    if host:                                   # last: without it the library still serves all but the microscaled calls
        if os.path.exists(HOST_TAG):
            os.remove(HOST_TAG)
        _link_host(host_obj.result())
        with open(HOST_TAG, "w") as f:
            f.write(_wanted_tag())
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
