"""Builds the gfx950 kernel library ``libxpu_graph_amd.so`` in-tree with hipcc, and on top of it
``libxpu_graph_amd_torch.so``, the torch ops that are implemented in C++ (host code).

    python -m xpu_graph_amd.build            # compile every csrc/*.hip and csrc/*.cpp and link

hipcc cross-compiles for gfx950 without a GPU.  Objects go to ``csrc/_obj``; the
shared library lands beside this file so that it travels with the source tree.
"""
import concurrent.futures
import os
import shutil
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
OBJ_DIR = os.path.join(CSRC, "_obj")
LIB_PATH = os.path.join(_HERE, "libxpu_graph_amd.so")
TORCH_OPS_PATH = os.path.join(_HERE, "libxpu_graph_amd_torch.so")

ARCH = "gfx950"
# Packed fp32 instructions are switched off for every device compile: the
# compiler otherwise forms them on its own from plain float code.
HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc_path():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the mi355x target needs the ROCm toolchain to build its kernels")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def host_compiler():
    """g++, or the clang++ that hipcc itself runs: what builds the kernels builds the torch ops."""
    clang = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")
    for cand in (shutil.which("g++"), shutil.which("clang++"), clang):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("no host C++ compiler found for torch_ops.cpp")


def _compile_torch_ops():
    """Object file of csrc/torch_ops.cpp: host code against the headers of the installed torch."""
    import torch

    root = os.path.join(os.path.dirname(torch.__file__), "include")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    obj = os.path.join(OBJ_DIR, "torch_ops.host.o")
    cmd = [
        host_compiler(), "-std=c++17", "-O2", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root}", f"-I{os.path.join(root, 'torch/csrc/api/include')}",
        f"-I{os.path.join(rocm, 'include')}", "-c", os.path.join(CSRC, "torch_ops.cpp"), "-o", obj,
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"the host compiler failed for torch_ops.cpp:\n{proc.stderr}")
    return obj


def _link_torch_ops(obj):
    import torch

    tmp = TORCH_OPS_PATH + ".tmp"
    cmd = [
        host_compiler(), "-shared", "-o", tmp, obj, f"-L{os.path.join(os.path.dirname(torch.__file__), 'lib')}", "-ltorch_cpu", "-ltorch", "-lc10",
        "-lc10_hip", f"-L{_HERE}", "-l:libxpu_graph_amd.so", "-Wl,-rpath,$ORIGIN",
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link of the torch ops failed:\n{proc.stderr}")
    os.replace(tmp, TORCH_OPS_PATH)


def _compile_one(src):
    obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-4] + ".o")
    cmd = [hipcc_path(), *HIPCC_FLAGS, "-c", src, "-o", obj]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{proc.stderr}")
    return obj


def build_library(verbose=True, jobs=None):
    """Compile every kernel source for gfx950 and link the C-ABI shared library, then the torch ops on top of it.

    The kernel library does not depend on the torch half: where that cannot be built (no headers, an error in it) the kernel
    library is in place all the same when the error is raised, without a torch half of another build beside it."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    wanted = {os.path.basename(s)[:-4] + ".o" for s in srcs} | {"torch_ops.host.o"}
    for stale in set(os.listdir(OBJ_DIR)) - wanted:
        os.remove(os.path.join(OBJ_DIR, stale))
    jobs = jobs or min(len(srcs) + 1, max(1, (os.cpu_count() or 2) - 1), 8)
    if verbose:
        print(f"[xpu_graph_amd.build] hipcc {ARCH}: {len(srcs)} sources, {jobs} jobs", flush=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as ex:
        torch_obj = ex.submit(_compile_torch_ops)
        objs = list(ex.map(_compile_one, srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc_path(), "-shared", "-fPIC", f"--offload-arch={ARCH}", "-o", tmp, *objs]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    try:
        _link_torch_ops(torch_obj.result())
    except (RuntimeError, OSError, ImportError) as e:
        if os.path.exists(TORCH_OPS_PATH):
            os.remove(TORCH_OPS_PATH)
        raise RuntimeError(f"{LIB_PATH} is built, the torch ops on top of it are not (their calls raise ImportError): {e}") from e
    if verbose:
        print(f"[xpu_graph_amd.build] wrote {LIB_PATH} and {TORCH_OPS_PATH}", flush=True)
    return LIB_PATH


if __name__ == "__main__":
    build_library()
    sys.exit(0)
