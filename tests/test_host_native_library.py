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
