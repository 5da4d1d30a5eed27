"""Builds csrc/*.cu into libkmb200.so (sm_100a) and csrc/torch_calls.cpp into _torch_calls.so, next to
this file.

    python -m sklearn_numba_dpex_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU.  Objects are rebuilt only when their source or a
header is newer, the extension also when the interpreter, torch or the command changed; the shared library links the CUDA runtime statically, so it has no
dependency on the interpreter's own CUDA libraries.
"""
import argparse
import concurrent.futures
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OBJ_DIR = os.path.join(CSRC, "build")
LIB_PATH = os.path.join(HERE, "libkmb200.so")
CALLS_PATH = os.path.join(HERE, "_torch_calls.so")
CALLS_STAMP = os.path.join(OBJ_DIR, "torch_calls.stamp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-v",
]


def _nvcc():
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the kmb200 library cannot be built")
    return path


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime():
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    paths += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return max(os.path.getmtime(p) for p in paths)


def _compile_one(nvcc, src, force, verbose):
    obj = os.path.join(OBJ_DIR, src[:-3] + ".o")
    src_path = os.path.join(CSRC, src)
    newest = max(os.path.getmtime(src_path), _headers_mtime())
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest:
        return obj, ""
    extra = os.environ.get("KMB_NVCC_EXTRA", "").split()
    cmd = [nvcc] + NVCC_FLAGS + extra + ["-I", INCLUDE, "-c", src_path, "-o", obj]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{proc.stdout}\n{proc.stderr}")
    log = proc.stderr if verbose else ""
    with open(obj[:-2] + ".ptxas.log", "w") as fh:
        fh.write(proc.stderr)
    return obj, log


def build(force=False, verbose=False):
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = _sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as pool:
        results = list(pool.map(lambda s: _compile_one(nvcc, s, force, verbose), srcs))
    objs = [r[0] for r in results]
    for _, log in results:
        if log:
            print(log)
    need_link = force or not os.path.exists(LIB_PATH) or any(
        os.path.getmtime(o) > os.path.getmtime(LIB_PATH) for o in objs)
    if need_link:
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB_PATH] + objs
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
    if importlib.util.find_spec("torch") is None:
        # an isolated build; one against some torch that pip fetches would not fit the one at run time
        print("torch is not installed where this build runs: the expert and 8-bit calls are left out. "
              "`pip install --no-build-isolation .` builds them with the torch that they will run with.")
    else:
        build_calls(force)
    return LIB_PATH


def build_calls(force=False):
    """The binding of the calls whose host time counts: a Python extension over torch's C++ tensors."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    src = os.path.join(CSRC, "torch_calls.cpp")
    includes = include_paths("cuda") + [sysconfig.get_paths()["include"], INCLUDE]
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DKMB_TORCH_VERSION="{torch.__version__}"',
           src, "-o", CALLS_PATH]
    cmd += [f"-I{path}" for path in includes] + [f"-L{path}" for path in library_paths("cuda")]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", f"-L{HERE}", "-l:libkmb200.so", "-Wl,-rpath,$ORIGIN"]
    # the extension fits one interpreter and one torch: an older file for others is no newer for its time
    made_for = "\n".join([sys.version, torch.__version__, *cmd])
    newest = max(os.path.getmtime(src), _headers_mtime())
    if not force and _calls_made_for() == made_for and os.path.exists(CALLS_PATH) and os.path.getmtime(CALLS_PATH) >= newest:
        return CALLS_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    if os.path.exists(CALLS_STAMP):
        os.remove(CALLS_STAMP)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on torch_calls.cpp:\n{proc.stdout}\n{proc.stderr}")
    with open(CALLS_STAMP, "w") as fh:
        fh.write(made_for)
    return CALLS_PATH


def _calls_made_for():
    """What the extension was built for and with, as build_calls noted it."""
    try:
        with open(CALLS_STAMP) as fh:
            return fh.read()
    except OSError:
        return None


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    sys.exit(0)
