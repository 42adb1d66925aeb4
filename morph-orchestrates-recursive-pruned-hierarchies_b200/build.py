"""Builds libmortar_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the torch
binding of the dense site's operators, _mortar_native.so, with the host compiler.

    python morph-orchestrates-recursive-pruned-hierarchies_b200/build.py [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libmortar_b200.so")
BINDING = os.path.join(CSRC, "torch_binding.cpp")
NATIVE = os.path.join(PKG, "_mortar_native.so")
SOURCES = ["host_pack.cpp", "prefill_sched.cpp", "stream_kernels.cu", "prefill_tc.cu", "stack_decode.cu",
           "router.cu", "backward.cu", "backward_tc.cu", "gemv_tc.cu", "layer_norm.cu", "dense_tc.cu", "fp8_quant.cu",
           "fp8_tc.cu", "dense_small.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


OBJ = os.path.join(PKG, "_build")            # per-source objects (ignored by git; only the .so is used)


def _deps_mtime(src: str) -> float:
    """A source is rebuilt when it, any header beside it or the public header is newer than its object."""
    paths = [os.path.join(CSRC, src), os.path.join(ROOT, "include", "mortar_b200.h")]
    paths += [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    return max(os.path.getmtime(p) for p in paths)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every source under csrc/ (in parallel, one object each) and link one shared library;
    returns its path."""
    from concurrent.futures import ThreadPoolExecutor
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    os.makedirs(OBJ, exist_ok=True)
    base = [nvcc, "-O3", "-std=c++17", "-lineinfo", *ARCH, "-Xcompiler", "-fPIC",
            "-I", os.path.join(ROOT, "include"), "-I", CSRC]
    if verbose:
        base += ["-Xptxas", "-v"]

    def compile_one(src: str):
        obj = os.path.join(OBJ, src + ".o")
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= _deps_mtime(src):
            return obj, False
        cmd = base + ["-c", os.path.join(CSRC, src), "-o", obj]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed ({res.returncode}): {' '.join(cmd)}")
        return obj, True

    with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        results = list(pool.map(compile_one, SOURCES))
    objs = [o for o, _ in results]
    if any(changed for _, changed in results) or not os.path.exists(LIB) or \
            os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        cmd = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", LIB]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError(f"link failed ({res.returncode}): {' '.join(cmd)}")
    build_binding(force=force, verbose=verbose)
    return LIB


BINDING_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_mortar_native"]
# The C++ runtime and the unwinder that torch runs on, whatever the compiler links by default: with copies of its own (a
# compiler that has only the static ones) the binding's exceptions end the process.  Compilers that do not know the first flag
# (g++ before 13) look into the shared library first all the same, since it comes before the one that they add.
NO_OWN_RUNTIME = "-nostdlib++"
RUNTIME = ["-l:libstdc++.so.6", "-shared-libgcc", "-l:libgcc_s.so.1"]


def build_binding(force: bool = False, verbose: bool = False):
    """Compiles csrc/torch_binding.cpp against the installed torch and links it to the library beside it;
    returns its path.  It is built again when a source is newer, or when the command, torch or Python
    are not those that it was built with.  Without torch or Python's headers it is left out (None): the library
    and its C entry points need neither."""
    import sysconfig
    python_include = sysconfig.get_paths()["include"]
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        missing = "torch is not installed"
    else:
        missing = None if os.path.exists(os.path.join(python_include, "Python.h")) else f"there is no Python.h in {python_include}"
    if missing:
        sys.stderr.write(f"{missing}: the torch binding of the dense site is not built, the C library is complete\n")
        return None
    cxx = os.environ.get("CXX", "g++")
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    include = [f"-isystem{d}" for d in cpp_extension.include_paths()]
    include += [f"-I{d}" for d in (python_include, os.environ.get("CUDA_HOME", "/usr/local/cuda") + "/include",
                                   os.path.join(ROOT, "include"))]
    knows = subprocess.run([cxx, NO_OWN_RUNTIME, "-E", "-x", "c++", os.devnull], capture_output=True).returncode == 0
    cmd = [cxx, *BINDING_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *include, BINDING, "-o", NATIVE, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           f"-L{PKG}", "-l:libmortar_b200.so", "-Wl,-rpath,$ORIGIN", *([NO_OWN_RUNTIME] if knows else []), *RUNTIME]
    made_with = "\n".join([*cmd, torch.__version__, str(sysconfig.get_config_var("SOABI"))])
    record = os.path.join(OBJ, "_mortar_native.built_with")
    newest = max(os.path.getmtime(f) for f in (BINDING, os.path.join(ROOT, "include", "mortar_b200.h")))
    if not force and os.path.exists(NATIVE) and os.path.getmtime(NATIVE) >= newest and os.path.exists(record):
        with open(record) as f:
            if f.read() == made_with:
                return NATIVE
    if os.path.exists(record):
        os.remove(record)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}): {' '.join(cmd)}")
    os.makedirs(OBJ, exist_ok=True)
    with open(record, "w") as f:
        f.write(made_with)
    return NATIVE


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
