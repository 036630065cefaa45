"""The C++ ops' library beside the kernel library: what the package does where it is missing or does not fit.  No GPU needed."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
import torch
from xpu_graph_amd import _lib

assert "xpu_graph_amd.ops" not in sys.modules
_lib.TORCH_OPS_PATH = sys.argv[1]
import xpu_graph_amd.ops

ops = torch.ops.xpu_ops
x, t = torch.empty(1, 2, 4, 64, device="meta"), torch.empty(4, 64, device="meta")
assert ops.rms_norm(x, t[0], 1e-6).shape == x.shape and ops.rope(x, t, t).shape == x.shape  # the other ops
assert ops.rope_axes(x, t, t, None, []).shape == x.shape
cuda = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
x, t = torch.zeros(1, 2, 4, 64), torch.zeros(4, 64)
for call in (
    lambda: ops.rope_axes.default.redispatch(cuda, x, t, t, None, []),
    lambda: ops.linear_attn.default.redispatch(cuda, x, x, x, t[0, :2], None, None, 1.0),
):
    try:
        call()
    except ImportError as e:
        assert sys.argv[1] in str(e) and "xpu_graph_amd.build" in str(e), e
        print("refused:", e)
    else:
        raise AssertionError("no error")
"""


def run(path):
    return subprocess.run([sys.executable, "-c", textwrap.dedent(PROGRAM), str(path)], cwd=ROOT, capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("kind", ["missing", "no library", "other symbols"])
def test_the_other_ops_do_not_need_it(tmp_path, kind):
    path = tmp_path / "libxpu_graph_amd_torch.so"
    if kind == "no library":
        path.write_bytes(b"built elsewhere")
    elif kind == "other symbols":  # as one built against another torch
        src = tmp_path / "x.cpp"
        src.write_text("void not_in_this_torch(); namespace { struct S { S() { not_in_this_torch(); } } s; }")
        subprocess.run(["g++", "-shared", "-fPIC", str(src), "-o", str(path)], check=True)
    done = run(path)
    assert done.returncode == 0, done.stderr
    assert done.stdout.count("refused:") == 2 and ("is missing" if kind == "missing" else "cannot be loaded") in done.stdout


@pytest.fixture
def small_tree(tmp_path, monkeypatch):
    """build.py on a tree of its own: one small kernel source, one small source of torch ops, an older build of both."""
    from xpu_graph_amd import build

    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "small.hip").write_text('extern "C" int xg_version(void) { return 100; }\n')
    (csrc / "torch_ops.cpp").write_text("#include <c10/util/Exception.h>\nint here() { return 1; }\n")
    for name, value in (("_HERE", ""), ("CSRC", "csrc"), ("OBJ_DIR", "csrc/_obj"), ("LIB_PATH", "libxpu_graph_amd.so"), ("TORCH_OPS_PATH", "libxpu_graph_amd_torch.so")):
        monkeypatch.setattr(build, name, str(tmp_path / value) if value else str(tmp_path))
    for path in (build.LIB_PATH, build.TORCH_OPS_PATH):
        with open(path, "w") as f:
            f.write("old")
    return build, csrc


def symbols(path):
    return subprocess.run(["nm", "-D", "--defined-only", path], capture_output=True, text=True, check=True).stdout


def test_the_kernel_library_is_built_before_the_torch_ops(small_tree):
    build, csrc = small_tree
    (csrc / "torch_ops.cpp").write_text("this is no C++\n")
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):
        build.build_library(verbose=False)
    assert "xg_version" in symbols(build.LIB_PATH)
    assert not os.path.exists(build.TORCH_OPS_PATH)  # none of another build is left beside it


def test_hipcc_alone_builds_both(small_tree, monkeypatch):
    build, _ = small_tree
    which = build.shutil.which
    monkeypatch.setattr(build.shutil, "which", lambda name, *a, **k: None if name in ("g++", "clang++") else which(name, *a, **k))
    build.build_library(verbose=False)
    assert "xg_version" in symbols(build.LIB_PATH) and "here" in symbols(build.TORCH_OPS_PATH)


def test_no_host_compiler_leaves_the_kernel_library(small_tree, monkeypatch):
    build, _ = small_tree

    def none():
        raise RuntimeError("no host C++ compiler found")

    monkeypatch.setattr(build, "host_compiler", none, raising=False)
    with pytest.raises(RuntimeError, match="no host C"):
        build.build_library(verbose=False)
    assert "xg_version" in symbols(build.LIB_PATH)
