"""Refusals of the query / key preparation ops: shapes through their Meta implementations, arguments of the C entry points
(checked before any launch), and the axis map.  No GPU needed."""
import ctypes

import pytest
import torch

from xpu_graph_amd import _lib
from xpu_graph_amd import ops as xops  # noqa: F401

OPS = torch.ops.xpu_ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize(
    "x,table,pos,sections,error",
    [
        ((2, 3, 64), (8, 64), None, [], ValueError),  # not [B, H, S, D]
        ((2, 3, 8, 24), (8, 24), None, [], ValueError),  # head dim
        ((2, 3, 8, 528), (8, 528), None, [], ValueError),  # head dim beyond the kernel
        ((2, 3, 8, 64), (7, 64), None, [], ValueError),  # rows for another length
        ((2, 3, 8, 64), (8, 48), None, [], ValueError),  # neither R nor R/2 columns
        ((2, 3, 8, 64), (2, 8, 64), None, [], ValueError),  # a table per batch entry
        ((2, 3, 8, 64), (9, 32), (2, 2, 8), [16], ValueError),  # two position rows for one axis
        ((2, 3, 8, 64), (9, 32), (2, 8), [16, 16], ValueError),  # several axes need [axes, B, S]
        ((2, 3, 8, 64), (9, 32), (3, 2, 8), [16, 16], ValueError),  # axes
        ((2, 3, 8, 64), (9, 32), (2, 3, 8), [16, 16], ValueError),  # batch
        ((2, 3, 8, 64), (9, 32), (2, 2, 9), [16, 16], ValueError),  # length
        ((2, 3, 8, 64), (8, 32), None, [16, 16], ValueError),  # several axes without positions
        ((2, 3, 8, 64), (9, 32), (2, 2, 8), [15, 16], ValueError),  # R no multiple of 16
        ((2, 3, 8, 64), (9, 40), (2, 2, 8), [20, 20], ValueError),  # R beyond the head dim
        ((2, 3, 8, 64), (9, 32), (2, 2, 8), [-8, 40], ValueError),
        ((2, 3, 8, 64), (9, 32), (5, 2, 8), [8, 8, 8, 4, 4], ValueError),  # five axes
        ((2, 3, 8, 64), (0, 32), (2, 2, 8), [16, 16], ValueError),  # an empty table
    ],
)
def test_rope_axes_refuses(x, table, pos, sections, error):
    p = meta(*pos, dtype=torch.int64) if pos else None
    t = meta(*table, dtype=torch.float32)
    with pytest.raises(error):
        OPS.rope_axes(meta(*x), t, t, p, sections)
    with pytest.raises(error):
        OPS.rope_axes_bwd(meta(*x), t, t, p, sections)


def test_types_and_weights_are_checked():
    x, t = meta(2, 3, 8, 64), meta(8, 64, dtype=torch.float32)
    with pytest.raises(TypeError):
        OPS.rope_axes(x, t.half(), t.half(), None, [])  # tables of another 16-bit type
    with pytest.raises(TypeError):
        OPS.rope_axes(x, t, t, meta(8, dtype=torch.int16), [])
    with pytest.raises(ValueError):
        OPS.rope_axes(x, t, meta(8, 32, dtype=torch.float32), None, [])
    args = (t, t, None, [], False, 1e-6)
    with pytest.raises(ValueError):
        OPS.qk_norm_rope(x, meta(2, 1, 9, 64), None, None, *args)
    with pytest.raises(ValueError):
        OPS.qk_norm_rope(x, x, meta(32), None, *args)
    with pytest.raises(TypeError):
        OPS.qk_norm_rope(x, x.half(), None, None, *args)
    oq, ok = OPS.qk_norm_rope(x, meta(2, 1, 8, 64), meta(64), None, *args)
    assert oq.shape == x.shape and ok.shape == (2, 1, 8, 64)
    dq, dk, gwq, gwk = OPS.qk_norm_rope_bwd(x, x, meta(64), None, x, x, *args, True)
    assert gwq.shape == (64,) and gwk.shape == (0,)


def test_layouts_survive():
    x = meta(2, 8, 3, 64).transpose(1, 2)
    t = meta(8, 32, dtype=torch.float32)
    assert OPS.rope_axes(x, t, t, None, []).stride() == x.stride()


def test_a_part_of_a_projection_gives_results_in_its_order():
    heads = meta(2, 3, 12 * 64).view(2, 3, 12, 64).transpose(1, 2)
    t = meta(3, 32, dtype=torch.float32)
    q, k = OPS.qk_norm_rope(heads[:, :8], heads[:, 8:10], None, None, t, t, None, [], False, 1e-6)
    assert q.stride() == (3 * 8 * 64, 64, 8 * 64, 1) and k.stride() == (3 * 2 * 64, 64, 2 * 64, 1)
    assert OPS.rope_axes(heads[:, :1].expand(2, 4, 3, 64), t, t, None, []).is_contiguous()  # shared heads: no order of their own


def test_layouts_of_dimensions_of_one_element():
    """What torch keeps as the stride of a dimension of size 1 does not decide about the layout."""
    x = torch.empty(1, 3, 8, 64, device="meta", dtype=torch.bfloat16).as_strided((1, 3, 8, 64), (1 << 40, 64, 192, 1))
    odd = torch.empty_strided((1, 3, 8, 64), (8 * 192 + 1, 64, 192, 1), device="meta", dtype=torch.bfloat16)
    t = meta(8, 32, dtype=torch.float32)
    for y in (x, odd):
        assert OPS.rope_axes(y, t, t, None, []).stride()[1:] == (64, 192, 1)


def test_the_gpu_implementations_are_built_and_loaded():
    assert _lib.torch_ops_built()
    for name in ("rope_axes", "rope_axes_bwd", "qk_norm_rope", "qk_norm_rope_bwd", "linear_attn", "linear_attn_bwd", "linear_attn_step"):
        for key in ("CUDA", "Autograd", "Meta"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key(f"xpu_ops::{name}", key), (name, key)


def test_cpu_tensors_have_no_kernel():
    x, t = torch.zeros(1, 1, 2, 64), torch.zeros(2, 32)
    with pytest.raises(NotImplementedError):
        OPS.rope_axes(x, t, t, None, [])


def test_entry_points_refuse_before_any_launch():
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) & ~15)
    S3 = ctypes.c_int64 * 3
    st = S3(512, 256, 64)

    def rotary(**kw):
        r = _lib.XgRotary(p, p, 9, 32, 32, 64)
        r.axes, r.table_dtype = 1, 2
        r.positions, r.positions_64bit = p, 1
        for name, value in kw.items():
            if name == "pos_strides":
                for i in range(3):
                    r.pos_strides[i] = value[i]
            else:
                setattr(r, name, value)
        return r

    def rope(B=2, H=2, S=4, D=64, xs=st, dtype=2, x=p, r=None, **kw):
        return lib.xg_rope_axes(x, p, B, H, S, D, xs, st, r if r is not None else rotary(**kw), 0, dtype, None)

    assert rope(B=0) == 0 and rope(S=0) == 0  # nothing to launch
    assert rope(dtype=3) == -1 and rope(table_dtype=1) == -1
    assert rope(D=24) == -2 and rope(D=528) == -2 and rope(B=-1) == -2
    assert rope(rot_dim=8) == -2 and rope(rot_dim=80) == -2 and rope(table_cols=48) == -2 and rope(table_stride=16) == -2
    assert rope(table_rows=0) == -2 and rope(positions=None, table_rows=3) == -2 and rope(positions=None, axes=2) == -2
    assert rope(axes=5) == -7 and rope(axes=0) == -7 and rope(axes=2) == -4  # an axis map is missing
    assert rope(axes=2, pair_axis=bytes([2] * 32)) == -7  # an axis that is not there
    assert rope(pos_strides=(0, -1, 1)) == -2
    assert rope(x=None) == -4 and rope(cos_table=None) == -4
    assert lib.xg_rope_axes(p, p, 2, 2, 4, 64, st, st, None, 0, 2, None) == -4
    assert rope(xs=S3(512, 250, 64)) == -3 and rope(xs=S3(512, -256, 64)) == -2 and rope(x=ctypes.c_void_p(p.value + 8)) == -3
    assert rope(table_stride=33) == -3 and rope(cos_table=p.value + 4) == -3 and rope(positions=p.value + 4) == -3
    assert rope(B=1 << 20, S=1 << 20) == -5  # more rows than a launch takes
    assert rope(B=1 << 30, H=1, S=1, D=128) == -5  # more threads

    def qk(H=2, Hkv=1, w_dtype=2, k=p, r=None):
        return lib.xg_qk_norm_rope(p, k, p, p, p, p, 2, H, Hkv, 4, 64, st, st, st, st, r or rotary(), 1e-6, 2, w_dtype, None)

    assert qk(H=0, Hkv=0) == 0 and qk(k=None) == -4 and qk(w_dtype=1) == -1 and qk(H=-1) == -2

    n = lib.xg_qk_norm_rope_bwd_workspace_floats(2, 2, 1, 4, 64)
    assert n > 0 and n % 64 == 0 and lib.xg_qk_norm_rope_bwd_workspace_floats(2, 2, 1, 4, 24) == 0

    def bwd(ws=p, ws_n=n, gq=p):
        return lib.xg_qk_norm_rope_bwd(p, p, p, p, gq, p, p, p, p, p, ws, ws_n, 2, 2, 1, 4, 64, st, st, st, st, st, st, rotary(), 1e-6, 2, 2, None)

    assert bwd(ws=None) == -4 and bwd(ws_n=n - 1) == -7 and bwd(gq=None) == -4
