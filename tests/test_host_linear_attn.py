"""Refusals of the linear attention ops: shapes through their Meta implementations, arguments of the C entry points (checked
before any launch).  No GPU needed."""
import ctypes

import pytest
import torch

from xpu_graph_amd import _lib
from xpu_graph_amd import ops as xops  # noqa: F401

OPS = torch.ops.xpu_ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def call(q=(2, 4, 8, 64), k=(2, 2, 8, 64), v=None, g=(4,), state=None, lengths=None, dtype=torch.bfloat16, g_dtype=torch.float32, n_dtype=torch.int64):
    s = meta(*state, dtype=torch.float32) if state else None
    n = meta(*lengths, dtype=n_dtype) if lengths else None
    return OPS.linear_attn(meta(*q, dtype=dtype), meta(*k, dtype=dtype), meta(*(v or k), dtype=dtype), meta(*g, dtype=g_dtype), s, n, 1.0)


def test_shapes():
    o, s = call()
    assert o.shape == (2, 4, 8, 64) and s.shape == (2, 4, 64, 64) and s.dtype == torch.float32
    o, s = call(state=(2, 4, 64, 64), lengths=(2,), dtype=torch.float16, n_dtype=torch.int32)
    assert o.dtype == torch.float16
    q, k = meta(2, 4, 8, 64), meta(2, 2, 8, 64)
    dq, dk, dv, ds = OPS.linear_attn_bwd(q, k, k, meta(4, dtype=torch.float32), None, None, q, None, 1.0, False)
    assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == k.shape and ds.numel() == 0


@pytest.mark.parametrize(
    "kw,error",
    [
        (dict(q=(2, 4, 64)), ValueError),
        (dict(k=(2, 3, 8, 64)), ValueError),  # 4 query heads over 3
        (dict(k=(2, 0, 8, 64)), ValueError),
        (dict(k=(2, 2, 9, 64)), ValueError),
        (dict(k=(1, 2, 8, 64)), ValueError),
        (dict(v=(2, 2, 8, 128)), ValueError),  # values of another width
        (dict(q=(2, 4, 8, 96), k=(2, 2, 8, 96)), ValueError),
        (dict(g=(2,)), ValueError),
        (dict(g_dtype=torch.bfloat16), ValueError),
        (dict(dtype=torch.float32), TypeError),
        (dict(state=(2, 2, 64, 64)), ValueError),
        (dict(state=(2, 4, 64, 128)), ValueError),
        (dict(lengths=(3,)), ValueError),
        (dict(lengths=(2,), n_dtype=torch.int16), ValueError),
    ],
)
def test_refuses(kw, error):
    with pytest.raises(error):
        call(**kw)


def test_backward_and_step_refuse():
    q, k, g = meta(2, 4, 8, 64), meta(2, 2, 8, 64), meta(4, dtype=torch.float32)
    with pytest.raises(ValueError):
        OPS.linear_attn_bwd(q, k, k, g, None, None, k, None, 1.0, False)
    with pytest.raises(ValueError):
        OPS.linear_attn_bwd(q, k, k, g, None, None, q, meta(2, 4, 64, 64), 1.0, False)  # a 16-bit state gradient
    s = meta(2, 4, 64, 64, dtype=torch.float32)
    with pytest.raises(ValueError):
        OPS.linear_attn_step(q, k, k, g, s, 1.0)  # eight tokens
    q, k = q[:, :, :1], k[:, :, :1]
    assert OPS.linear_attn_step(q, k, k, g, s, 1.0).shape == q.shape
    with pytest.raises(ValueError):
        OPS.linear_attn_step(q, k, k, g, s.transpose(2, 3), 1.0)


def test_entry_points_refuse_before_any_launch():
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) & ~15)
    off = ctypes.c_void_p(p.value + 8)
    S3, S2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
    st = S3(1 << 14, 1 << 12, 64)
    need = lib.xg_linear_attn_workspace_floats(1, 2, 1024, 64)
    assert need > 0 and need % 4096 == 0
    assert lib.xg_linear_attn_workspace_floats(1, 2, 64, 64) == 0 and lib.xg_linear_attn_workspace_floats(1, 2, 1024, 96) == 0

    def fwd(q=p, g=p, state=None, n=None, out=p, ws=p, ws_n=need, B=1, H=2, Hkv=2, S=1024, D=64, qs=st, scale=1.0, dtype=2):
        return lib.xg_linear_attn(q, p, p, g, state, n, 1, out, p, ws, ws_n, B, H, Hkv, S, D, qs, st, st, st, scale, dtype, None)

    assert fwd(B=0) == 0 and fwd(S=0) == 0 and fwd(H=0, Hkv=0) == 0
    assert fwd(dtype=0) == -1 and fwd(D=96) == -2 and fwd(S=-1) == -2 and fwd(H=3) == -2 and fwd(Hkv=0) == -2
    assert fwd(q=None) == -4 and fwd(g=None) == -4 and fwd(out=None) == -4 and fwd(ws=None) == -4 and fwd(ws_n=need - 1) == -7
    assert fwd(q=off) == -3 and fwd(state=off) == -3 and fwd(qs=S3(1, 2, 3)) == -3 and fwd(qs=S3(-8, 8, 8)) == -2
    assert fwd(n=ctypes.c_void_p(p.value + 4)) == -3
    assert fwd(qs=S3(1 << 14, 1 << 12, 1 << 26)) == -5  # tokens too far apart for 32-bit offsets within a chunk
    assert fwd(scale=float("nan")) == -7 and fwd(scale=float("inf")) == -7 and fwd(B=1 << 20, H=2) == -5

    need_b = lib.xg_linear_attn_bwd_workspace_floats(1, 2, 1, 1024, 64)
    assert need_b == 3 * need + 2 * 2 * 1024 * 64

    def bwd(do=p, dq=p, ws=p, ws_n=need_b):
        return lib.xg_linear_attn_bwd(p, p, p, p, None, None, 0, do, None, dq, p, p, None, ws, ws_n, 1, 2, 1, 1024, 64, *[st] * 7, 1.0, 2, None)

    assert bwd(do=None) == -4 and bwd(dq=None) == -4 and bwd(dq=off) == -3 and bwd(ws=None) == -4 and bwd(ws_n=need_b - 1) == -7

    def step(state=p, ss=(2 * 4096, 4096), B=2, H=2, D=64):
        return lib.xg_linear_attn_step(p, p, p, p, state, p, B, H, H, D, *[S2(128, 64)] * 4, S2(*ss), 1.0, 2, None)

    assert step(B=0) == 0 and step(state=None) == -4 and step(D=32) == -2 and step(state=off) == -3 and step(ss=(8192, 4098)) == -3
    assert step(ss=(0, 4096)) == -2 and step(ss=(8192, 0)) == -2 and step(ss=(4096, 4096)) == -2  # states that overlap


def test_key_heads_without_query_heads():
    q, k = meta(2, 0, 8, 64), meta(2, 3, 8, 64)
    dq, dk, dv, _ = OPS.linear_attn_bwd(q, k, k, meta(0, dtype=torch.float32), None, None, q, None, 1.0, False)
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) & ~15)
    off = ctypes.c_void_p(p.value + 8)
    st = (ctypes.c_int64 * 3)(1 << 14, 1 << 12, 64)

    def bwd(dk=p, dv=p, B=2, Hkv=3, S=8, D=64, s=st):
        return lib.xg_linear_attn_bwd(*[None] * 6, 0, None, None, None, dk, dv, p, None, 0, B, 0, Hkv, S, D, *[st] * 5, s, s, 1.0, 2, None)

    assert bwd(B=0) == 0 and bwd(S=0) == 0 and bwd(Hkv=0) == 0  # nothing to write
    assert bwd(dk=None) == -4 and bwd(dv=None) == -4 and bwd(dk=off) == -3 and bwd(s=None) == -4
    assert bwd(D=96) == -2 and bwd(Hkv=1 << 40) == -5 and bwd(s=(ctypes.c_int64 * 3)(1, 2, 3)) == -3


def test_states_that_share_memory_are_refused():
    """Workgroups of one launch read the states that come in while others write the one that goes out."""
    lib = _lib.lib()
    B, H, S, D = 1, 2, 64, 64
    buf = ctypes.create_string_buffer(1 << 17)
    base = (ctypes.addressof(buf) + 15) & ~15
    p = ctypes.c_void_p(base)
    at = lambda floats: ctypes.c_void_p(base + 4 * floats)  # noqa: E731
    half, whole = D * D, H * D * D

    short = (ctypes.c_int64 * 3)(1 << 14, 1 << 12, 4)  # what passes the states is refused for its strides

    def fwd(state, state_out, S=S):
        return lib.xg_linear_attn(p, p, p, p, state, None, 0, p, state_out, None, 0, B, H, H, S, D, *[short] * 4, 1.0, 2, None)

    def bwd(state, d_state_out, d_state, S=S):
        return lib.xg_linear_attn_bwd(p, p, p, p, state, None, 0, p, d_state_out, p, p, p, d_state, None, 0, B, H, H, S, D, *[short] * 7, 1.0, 2, None)

    assert fwd(p, p) == -3 and fwd(p, at(whole)) == -3 and fwd(at(whole), p) == -3 and fwd(None, p) == -3 and fwd(p, None) == -3
    for n in (S, 0):
        assert fwd(p, at(half), n) == -7 and fwd(at(half), p, n) == -7 and bwd(None, p, at(half), n) == -7
    assert bwd(p, None, p) == -7 and bwd(None, p, p) == -7 and bwd(at(half), None, p) == -7
    assert bwd(p, p, at(whole)) == -3 and bwd(p, p, None) == -3 and bwd(None, None, p) == -3
    assert bwd(None, p, p, 0) == 0 and bwd(p, None, None, 0) == 0  # nothing is computed: the gradient is where it belongs
