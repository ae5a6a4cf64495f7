"""Builds the CUDA backend (libphoenix_core_b200.so) for sm_100a, in-tree, with nvcc.

Every source is compiled to an object file of its own (in parallel, and only when it or a header is newer than
the object), then the objects are linked into one shared library next to the sources.

The extension module through which Python calls the block operators (binding.cpp, against torch's headers) is built next to the package's modules.

Usage: python -m phoenix_core_b200.csrc.build [--force] [--verbose]
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libphoenix_core_b200.so")
OBJ_DIR = os.path.join(HERE, "build")
SOURCES = ["api.cu", "simt_qgemm.cu", "tensor_path.cu", "pointwise_tc.cu", "pointwise2_tc.cu", "pointwise8_tc.cu", "conv_tc.cu", "narrow_tc.cu",
           "conv_tf32.cu", "qgemm_tc.cu", "aux_bn.cu", "probe.cu", "dense8_quant.cu", "dense8_tc.cu", 
           "residual_norm.cu", "residual_norm_f32.cu", "residual_norm_f16.cu", "residual_norm_bf16.cu", "distill.cu"]
HEADERS = ["common.cuh", "tensor_path.cuh", "dense8.cuh", "residual_norm.h", "residual_norm.cuh", "packed.cuh", "e4m3.cuh", "umma.cuh", "tc_common.cuh", "unaligned_chunk.h", "column_halves.h", "sm_share.h", "class_shares.h", os.path.join("..", "..", "include", "phoenix_core_b200.h")]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
]


BINDING_SOURCE = os.path.join(HERE, "binding.cpp")
BINDING = os.path.join(os.path.dirname(HERE), "_binding.so")


def build_binding(force=False):
    """Compiles binding.cpp into phoenix_core_b200/_binding.so (host code: g++, torch's headers and libraries)."""
    if not force and _mtime(BINDING) >= max(_mtime(BINDING_SOURCE), _mtime(os.path.join(HERE, "build.py"))):
        return BINDING
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include"),
                sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    for i in includes:
        cmd += ["-isystem", i]
    cmd += ["-o", BINDING, BINDING_SOURCE, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("building %s failed" % BINDING)
    return BINDING


def _mtime(path):
    return os.path.getmtime(path) if os.path.exists(path) else 0.0


def _sources():
    return [s for s in SOURCES if os.path.exists(os.path.join(HERE, s))]


def _compile(nvcc, src, obj, verbose):
    cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", obj, src]
    return src, subprocess.run(cmd, cwd=HERE, capture_output=True, text=True)


def build(force=False, verbose=False):
    """Compiles every CUDA source of the backend into one shared library next to the sources."""
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJ_DIR, exist_ok=True)
    build_binding(force)
    newest_header = max([_mtime(os.path.join(HERE, h)) for h in HEADERS] + [_mtime(os.path.join(HERE, "build.py"))])
    todo = []
    objs = []
    for src in _sources():
        obj = os.path.join(OBJ_DIR, src[:-3] + ".o")
        objs.append(obj)
        if force or _mtime(obj) < max(_mtime(os.path.join(HERE, src)), newest_header):
            todo.append((src, obj))
    if todo:
        with ThreadPoolExecutor(max_workers=min(len(todo), os.cpu_count() or 1)) as pool:
            results = list(pool.map(lambda so: _compile(nvcc, so[0], so[1], verbose), todo))
        failed = [(s, r) for s, r in results if r.returncode != 0]
        for s, r in results:
            if r.returncode != 0 or verbose:
                sys.stderr.write("== %s\n%s%s" % (s, r.stdout, r.stderr))
        if failed:
            raise RuntimeError("nvcc failed building " + ", ".join(s for s, _ in failed))
    if todo or not os.path.exists(LIB) or any(_mtime(o) > _mtime(LIB) for o in objs):
        res = subprocess.run([nvcc, "-shared", "-o", LIB] + objs, cwd=HERE, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("linking libphoenix_core_b200.so failed")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
