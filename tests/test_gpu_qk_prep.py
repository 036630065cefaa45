"""Query / key preparation on the GPU: rotary positions with several axes (xpu_ops::rope_axes) and the per-head norm with
rotation (xpu_ops::qk_norm_rope), forward and gradients, against the formulas in 64 bits.

Tolerances: the kernels compute in fp32 and round once, so a result is off by at most half a step of its type at the exact
value, plus the fp32 chain in front of that rounding.  The chain of one element is a row sum (at most 16 sequential terms per
lane and 5 tree steps), rsqrt, three products and the two products and the sum of the rotation: under 32 roundings of 2^-24,
each of at most the magnitude of the terms that are added."""
import pytest
import torch

from xpu_graph_amd import HIPGraphRunner

pytestmark = pytest.mark.gpu

CHAIN = 32 * 2.0**-24


def _xops():
    import xpu_graph_amd.ops as xops

    return xops


def _ops():
    _xops()
    return torch.ops.xpu_ops


def assert_rounded_once(got, want, magnitude, what, chain=CHAIN):
    """|got - want| <= half a step of got's type at want + chain * magnitude (+ half a subnormal step)."""
    info = torch.finfo(got.dtype)
    half = 0.0 if got.dtype == torch.float32 else info.eps / 2
    tol = want.abs() * half * (1 + 2.0**-8) + chain * magnitude + info.smallest_normal * info.eps
    err = (got.double() - want).abs()
    worst = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def tables(rows, cols, device, dtype, seed, full):
    """cos / sin of random angles [rows, cols]; full: two independent halves (what a rotation by real angles never has, so
    that a swapped half shows)."""
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(rows, cols * (2 if full else 1), generator=g, dtype=torch.float64) * 6.28
    return angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device)


def pair_axes(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n = len(sections)
    return [i % n if i < n * sections[i % n] else 0 for i in range(sum(sections))]


def angles(cos, sin, positions, sections, interleaved, B, S, R):
    """(c_lo, c_hi, s_lo, s_hi), each [B, 1, S, R/2] in 64 bits."""
    half = R // 2
    axis = torch.tensor(pair_axes(sections, interleaved) if sections else [0] * half, device=cos.device)
    pair = torch.arange(half, device=cos.device)
    if positions is None:
        at = torch.arange(S, device=cos.device).view(1, S, 1).expand(B, S, half)
        at = at if cos.shape[0] > 1 else torch.zeros_like(at)
    else:
        pos = positions.long().reshape((1,) * (3 - positions.dim()) + tuple(positions.shape)).expand(max(len(sections), 1), B, S)
        at = pos[axis].permute(1, 2, 0)
    hi = pair + (half if cos.shape[-1] == R else 0)
    return tuple(t.double()[at, col][:, None] for t in (cos, sin) for col in (pair, hi))


def turn(n, ang, R):
    c1, c2, s1, s2 = ang
    a, b = n[..., : R // 2], n[..., R // 2 : R]
    y = torch.cat([a * c1 - b * s1, b * c2 + a * s2, n[..., R:]], -1)
    mag = torch.cat([(a * c1).abs() + (b * s1).abs(), (b * c2).abs() + (a * s2).abs(), n[..., R:].abs()], -1)
    return y, mag


def turn_back(g, ang, R):
    c1, c2, s1, s2 = ang
    a, b = g[..., : R // 2], g[..., R // 2 : R]
    y = torch.cat([a * c1 + b * s2, b * c2 - a * s1, g[..., R:]], -1)
    mag = torch.cat([(a * c1).abs() + (b * s2).abs(), (b * c2).abs() + (a * s1).abs(), g[..., R:].abs()], -1)
    return y, mag


def norm64(x, eps):
    x = x.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return x * r, r


def make(B, H, S, D, dtype, device, seed, layout="bshd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "bhsd":
        return torch.randn(B, H, S, D, generator=g).to(dtype).to(device)
    return torch.randn(B, S, H, D, generator=g).to(dtype).to(device).transpose(1, 2)


def make_positions(kind, axes, B, S, P, device, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "none":
        return None
    shape = {"s": (S,), "bs": (B, S), "abs": (axes, B, S), "a1s": (axes, 1, S)}[kind]
    pos = torch.randint(0, P, shape, generator=g)
    pos.view(-1)[:2] = torch.tensor([0, P - 1])[: pos.numel()]  # both ends of the table
    return pos.to(device)


# head dim, rotated columns, sections, woven, positions, table columns per pair (1) or per element (2), layout
CASES = [
    (16, 16, [], False, "none", 2, "bhsd"),
    (64, 64, [], False, "bs", 1, "bshd"),
    (64, 32, [16], False, "s", 2, "bshd"),
    (80, 80, [], False, "bs", 1, "bshd"),
    (96, 48, [8, 8, 8], False, "abs", 1, "bhsd"),
    (128, 128, [16, 24, 24], False, "abs", 1, "bshd"),
    (128, 128, [24, 20, 20], True, "abs", 2, "bshd"),
    (128, 64, [5, 11, 16], True, "a1s", 1, "bhsd"),
    (128, 128, [7, 0, 30, 27], False, "abs", 1, "bshd"),
    (256, 256, [64, 64], True, "abs", 2, "bshd"),
    (512, 512, [], False, "bs", 1, "bshd"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=[f"d{c[0]}r{c[1]}a{len(c[2]) or 1}{'w' if c[3] else ''}" for c in CASES])
def test_rope_axes_and_its_transpose(device, dtype, case):
    D, R, sections, woven, kind, per, layout = case
    for B, H, S in ((1, 1, 1), (2, 3, 37)):
        P = 50
        x = make(B, H, S, D, dtype, device, 1 + S, layout)
        cos, sin = tables(P if kind != "none" else S, R // 2, device, torch.float32, 2, per == 2)
        pos = make_positions(kind, max(len(sections), 1), B, S, P, device, 3)
        for t_dtype in {dtype, torch.float32}:
            c, s = cos.to(t_dtype), sin.to(t_dtype)
            ang = angles(c, s, pos, sections, woven, B, S, R)
            got = _ops().rope_axes(x, c, s, pos, sections, woven)
            assert got.shape == x.shape and got.dtype == dtype and got.stride() == x.stride()
            assert_rounded_once(got, *turn(x.double(), ang, R), "rope_axes")
            got = _ops().rope_axes_bwd(x, c, s, pos.int() if pos is not None else None, sections, woven)
            assert_rounded_once(got, *turn_back(x.double(), ang, R), "rope_axes_bwd")


def check_qk(device, dtype, case, B, H, Hkv, S, weights, seed=1, packed=False):
    D, R, sections, woven, kind, per, layout = case
    P, eps = 60, 1e-6
    if packed:
        heads = make(B, H + 2 * Hkv, S, D, dtype, device, seed)
        q, k = heads[:, :H], heads[:, H : H + Hkv]
    else:
        q, k = make(B, H, S, D, dtype, device, seed, layout), make(B, Hkv, S, D, dtype, device, seed + 1, layout)
    q, k = q * 3, k * 0.2  # a norm that does nothing would show
    cos, sin = tables(P if kind != "none" else S, R // 2, device, torch.float32, 2, per == 2)
    pos = make_positions(kind, max(len(sections), 1), B, S, P, device, 3)
    g = torch.Generator().manual_seed(seed + 7)
    w_dtype = torch.float32 if weights == "fp32" else dtype
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(w_dtype).to(device) for _ in range(2)) if weights != "none" else (None, None)
    ang = angles(cos, sin, pos, sections, woven, B, S, R)
    args = (cos, sin, pos, sections, woven, eps)
    oq, ok = _ops().qk_norm_rope(q, k, wq, wk, *args)
    gq, gk = make(B, H, S, D, dtype, device, seed + 3), make(B, Hkv, S, D, dtype, device, seed + 4)
    dq, dk, gwq, gwk = _ops().qk_norm_rope_bwd(q, k, wq, wk, gq, gk, *args, True)
    for x, w, o, gy, dx, gw in ((q, wq, oq, gq, dq, gwq), (k, wk, ok, gk, dk, gwk)):
        assert o.shape == x.shape and dx.shape == x.shape and o.dtype == dtype and dx.dtype == dtype
        xhat, r = norm64(x, eps)
        w64 = w.double() if w is not None else torch.ones(D, device=device, dtype=torch.float64)
        assert_rounded_once(o, *turn(xhat * w64, ang, R), "qk_norm_rope")
        gn, gn_mag = turn_back(gy.double(), ang, R)
        dot = (gn * w64 * xhat).mean(-1, keepdim=True)
        dot_mag = (gn_mag * (w64 * xhat).abs()).mean(-1, keepdim=True)
        assert_rounded_once(dx, r * (gn * w64 - xhat * dot), r * (gn_mag * w64.abs() + xhat.abs() * dot_mag), "qk_norm_rope_bwd")
        if w is None:
            assert gw.numel() == 0
            continue
        assert gw.shape == w.shape and gw.dtype == w.dtype
        # the sum over rows: at most rows / 512 + 2 terms a lane, 256 rows a block, 16 + 64 partial rows
        depth = 340 + B * S * x.shape[1] / 512
        assert_rounded_once(gw, (gn * xhat).sum((0, 1, 2)), (gn_mag * xhat.abs()).sum((0, 1, 2)), "weight gradient", CHAIN + depth * 2.0**-24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=[f"d{c[0]}r{c[1]}a{len(c[2]) or 1}{'w' if c[3] else ''}" for c in CASES])
@pytest.mark.parametrize("weights", ["own", "fp32", "none"])
def test_qk_norm_rope_and_its_gradients(device, dtype, case, weights):
    check_qk(device, dtype, case, 2, 6, 2, 23, weights)


@pytest.mark.parametrize("B,H,Hkv,S", [(1, 1, 1, 1), (3, 7, 7, 1), (1, 5, 1, 257), (2, 9, 3, 1000), (4, 16, 4, 700)])
def test_qk_norm_rope_sizes_and_packed_projections(device, B, H, Hkv, S):
    check_qk(device, torch.bfloat16, CASES[5], B, H, Hkv, S, "own", packed=True)


def test_a_batch_of_many_heads_takes_the_grouped_path(device):
    check_qk(device, torch.bfloat16, CASES[1], 2, 30, 7, 4001, "own", packed=True)  # four heads a thread, a group that ends early


@pytest.mark.parametrize("case,S", [(CASES[1], 3001), (CASES[4], 2001), (CASES[6], 2001), (CASES[6], 6001)])
def test_two_and_four_heads_a_thread(device, case, S):
    check_qk(device, torch.bfloat16, case, 2, 9, 3, S, "own")  # (groups of the last odd head)


@pytest.mark.parametrize("case,S", [(CASES[6], 1501), (CASES[6], 6001), (CASES[4], 6001), (CASES[2], 9001)])
def test_two_and_eight_heads_a_thread(device, case, S):
    D, R, sections, woven, kind, per, _ = case
    B, H, P = 2, 11, 70
    x = make(B, H + 2, S, D, torch.float16, device, 5)[:, 1:-1]  # a part of something else
    cos, sin = tables(P if kind != "none" else S, R // 2, device, torch.float32, 2, per == 2)
    pos = make_positions(kind if kind != "s" else "bs", max(len(sections), 1), B, S, P, device, 3)
    ang = angles(cos, sin, pos, sections, woven, B, S, R)
    assert_rounded_once(_ops().rope_axes(x, cos, sin, pos, sections, woven), *turn(x.double(), ang, R), "rope_axes")
    assert_rounded_once(_ops().rope_axes_bwd(x, cos, sin, pos, sections, woven), *turn_back(x.double(), ang, R), "rope_axes_bwd")


def test_extreme_rows(device):
    """A row of zeros normalises to zeros; the largest and the smallest values of the type do not overflow in fp32."""
    D, eps = 64, 1e-6
    q = torch.zeros(1, 1, 4, D, device=device, dtype=torch.bfloat16)
    q[0, 0, 1] = 1e18
    q[0, 0, 2] = 2.0**-120
    q[0, 0, 3, 5] = -3.0
    cos, sin = tables(4, D // 2, device, torch.float32, 1, False)
    w = torch.ones(D, device=device, dtype=torch.bfloat16)
    oq, ok = _ops().qk_norm_rope(q, q, w, None, cos, sin, None, [], False, eps)
    want, mag = turn(norm64(q, eps)[0], angles(cos, sin, None, [], False, 1, 4, D), D)
    assert_rounded_once(oq, want, mag, "extreme rows")
    assert torch.equal(oq, ok) and (oq[0, 0, 0] == 0).all()


def test_a_position_outside_the_tables_gives_nan_and_touches_nothing_else(device):
    x = make(1, 2, 5, 64, torch.bfloat16, device, 1)
    cos, sin = tables(10, 16, device, torch.float32, 2, False)
    good = torch.tensor([[[0, 1, 2, 3, 4]], [[9, 8, 7, 6, 5]]], device=device)
    bad = good.clone()
    bad[1, 0, 2], bad[1, 0, 4] = 10, -1
    want, got = (_ops().rope_axes(x, cos, sin, p, [8, 8]) for p in (good, bad))
    hurt = torch.zeros(5, 64, dtype=torch.bool, device=device)
    for t in (2, 4):
        hurt[t, 8:16] = hurt[t, 24:32] = True  # the pairs of axis 1
    assert torch.isnan(got[:, :, hurt]).all() and torch.equal(got[:, :, ~hurt], want[:, :, ~hurt])


@pytest.mark.parametrize("per_element", [False, True])
def test_a_position_outside_one_axis_gives_nan_in_its_row(device, per_element):
    x, g = make(1, 2, 5, 64, torch.bfloat16, device, 1), make(1, 2, 5, 64, torch.bfloat16, device, 2)
    cos, sin = tables(10, 16, device, torch.float32, 2, per_element)
    good = torch.tensor([0, 1, 2, 3, 9], device=device)
    bad = torch.tensor([0, 10, 2, -(2**40), 9], device=device)
    want, got = (_ops().rope_axes(x, cos, sin, p, [16]) for p in (good, bad))
    out = torch.tensor([1, 3], device=device)
    assert torch.isnan(got[:, :, out, :32]).all() and torch.equal(got[:, :, out, 32:], x[:, :, out, 32:])
    kept = torch.tensor([0, 2, 4], device=device)
    assert torch.equal(got[:, :, kept], want[:, :, kept])
    args = lambda p: (x, x, None, None, g, g, cos, sin, p, [16], False, 1e-6, False)  # noqa: E731
    want, got = (_ops().qk_norm_rope_bwd(*args(p))[0] for p in (good, bad))
    assert torch.isnan(got[:, :, out]).all() and torch.equal(got[:, :, kept], want[:, :, kept])


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_agrees_with_the_norm_and_the_rotation_in_sequence(device, D, dtype):
    """rms_norm, then rope: the same but for the rounding of the normalised row between them.  That rounding is off by at most
    eps / 2 of each factor (mag adds their magnitudes up), the two results' own by eps / 2 of each; fp32 sums of D <= 128 squares
    and the products stay below 128 * 2^-24 < 1e-5 of mag."""
    q, k = make(2, 8, 300, D, dtype, device, D), make(2, 2, 300, D, dtype, device, D + 1)
    cos, sin = tables(300, D // 2, device, dtype, 5, True)
    g = torch.Generator().manual_seed(9)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype).to(device) for _ in range(2))
    half = torch.finfo(dtype).eps / 2
    for x, w, o in zip((q, k), (wq, wk), _ops().qk_norm_rope(q, k, wq, wk, cos, sin, None, [], False, 1e-6)):
        n = _ops().rms_norm(x, w, 1e-6)
        want = _ops().rope(n, cos, sin).double()
        mag = turn(n.double(), angles(cos, sin, None, [], False, 2, 300, D), D)[1]
        # (1 + half: the bounds are relative to unrounded values; the tiny term: fp16's subnormals)
        bound = (1 + 2 * half) * (half * mag + half * (o.double().abs() + want.abs()) + 1e-5 * mag) + 3 * 2.0**-25
        assert ((o.double() - want).abs() <= bound).all()


def test_one_axis_without_positions_equals_rope(device):
    x = make(2, 4, 33, 128, torch.bfloat16, device, 3)  # (fp16: the compiler may fuse a last product and its rounding differently per kernel)
    cos, sin = tables(33, 64, device, torch.bfloat16, 4, True)
    assert torch.equal(_ops().rope_axes(x, cos, sin, None, []), _ops().rope(x, cos, sin))
    row = cos[7:8], sin[7:8]
    assert torch.equal(_ops().rope_axes(x, *row, None, []), _ops().rope(x, *row))
    assert torch.equal(_ops().rope_axes(x, cos[None, None], sin[None, None], torch.arange(33, device=device), []), _ops().rope(x, cos, sin))


def test_odd_strides_are_copied_and_empty_inputs_return(device):
    base = torch.randn(2, 3, 9, 64 + 3, device=device).bfloat16()
    x = base[..., 1:65]  # a pitch and an offset that are no multiples of 16 bytes
    cos, sin = tables(9, 32, device, torch.float32, 1, False)
    assert torch.equal(_ops().rope_axes(x, cos, sin, None, []), _ops().rope_axes(x.contiguous(), cos, sin, None, []))
    one = x[:, :1].expand(2, 3, 9, 64)  # shared heads
    assert torch.equal(_ops().rope_axes(one, cos, sin, None, []), _ops().rope_axes(one.contiguous(), cos, sin, None, []))
    wide = torch.randn(9, 37, device=device)
    c2, s2 = wide[:, 1:33], wide[:, 4:36]  # unaligned table views
    assert torch.equal(_ops().rope_axes(x, c2, s2, None, []), _ops().rope_axes(x, c2.contiguous(), s2.contiguous(), None, []))
    for shape in ((0, 3, 9, 64), (2, 0, 9, 64), (2, 3, 0, 64)):
        e = torch.empty(shape, device=device, dtype=torch.bfloat16)
        t = tables(max(shape[2], 1), 32, device, torch.float32, 1, False)
        assert _ops().rope_axes(e, *t, None, []).shape == e.shape
    q, k = torch.empty(1, 2, 0, 64, device=device), torch.empty(1, 1, 0, 64, device=device)
    w = torch.ones(64, device=device)
    dq, dk, gwq, gwk = _ops().qk_norm_rope_bwd(q, k, w, w, q, k, *tables(1, 32, device, torch.float32, 1, False), None, [], False, 1e-6, True)
    assert dq.shape == q.shape and (gwq == 0).all() and (gwk == 0).all()


def test_gradients_through_autograd_and_against_differences(device):
    """torch.autograd on the ops, and central differences of the fp32 forward along random directions: with step h the
    difference of two sums of N outputs is off by about sqrt(N) 2^-23 / h from rounding and h^2 times the third derivative."""
    _xops().enable_autograd()
    B, H, Hkv, S, D, eps = 1, 3, 1, 7, 64, 1e-5
    cos, sin = tables(20, D // 2, device, torch.float32, 3, False)
    pos = make_positions("abs", 2, B, S, 20, device, 4)
    leaves = [make(B, H, S, D, torch.float32, device, 1), make(B, Hkv, S, D, torch.float32, device, 2)]
    leaves += [1 + 0.2 * torch.randn(D, device=device), 1 + 0.2 * torch.randn(D, device=device)]
    leaves = [t.requires_grad_() for t in leaves]
    up = [make(B, h, S, D, torch.float32, device, 9 + h) for h in (H, Hkv)]

    def forward(q, k, wq, wk):
        return _ops().qk_norm_rope(q, k, wq, wk, cos, sin, pos, [12, 20], True, eps)

    grads = torch.autograd.grad(forward(*leaves), leaves, up)
    h = 2.0**-6
    for i, leaf in enumerate(leaves):
        d = torch.randn_like(leaf)
        both = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * h * d if j == i else 0) for j, t in enumerate(leaves)]
            both.append(sum((o.double() * u.double()).sum() for o, u in zip(forward(*moved), up)))
        slope = ((both[0] - both[1]) / (2 * h)).item()
        want = (grads[i].double() * d.double()).sum().item()
        n = sum(u.numel() for u in up)
        assert abs(slope - want) <= n**0.5 * (2.0**-22 / h + 4 * h * h), (i, slope, want)
    x = leaves[0]
    y = _ops().rope_axes(x, cos, sin, pos, [12, 20], True)
    (gx,) = torch.autograd.grad(y, x, up[0])
    # the rotation is orthogonal: <y, up> = <x, gx>
    assert abs(((y.double() * up[0].double()).sum() - (x.double() * gx.double()).sum()).item()) <= x.numel() * 2.0**-20
    with pytest.raises(NotImplementedError):
        _ops().rope_axes(x, cos.clone().requires_grad_(), sin, pos, [12, 20], True).sum().backward()


def test_only_one_output_or_one_weight_takes_part(device):
    _xops().enable_autograd()
    q, k = make(1, 2, 5, 64, torch.bfloat16, device, 1).requires_grad_(), make(1, 1, 5, 64, torch.bfloat16, device, 2)
    w = torch.ones(64, device=device, dtype=torch.bfloat16).requires_grad_()
    t = tables(5, 32, device, torch.float32, 1, False)
    oq, _ = _ops().qk_norm_rope(q, k, w, None, *t, None, [], False, 1e-6)
    gq, gw = torch.autograd.grad(oq.sum(), (q, w))  # an expanded upstream gradient, no gradient for k
    want = _ops().qk_norm_rope_bwd(q, k, w, None, torch.ones_like(oq), torch.zeros_like(k), *t, None, [], False, 1e-6, True)
    assert torch.equal(gq, want[0]) and torch.equal(gw, want[2])


def test_results_do_not_depend_on_the_run(device):
    first = None
    for _ in range(3):
        q, k = make(2, 8, 513, 128, torch.bfloat16, device, 1), make(2, 8, 513, 128, torch.bfloat16, device, 2)
        w = torch.ones(128, device=device)
        out = _ops().qk_norm_rope_bwd(q, k, w, w, q, k, *tables(513, 64, device, torch.float32, 1, False), None, [], False, 1e-6, True)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_side_stream_and_graph_replays(device):
    cos, sin = tables(64, 32, device, torch.float32, 3, False)
    w = torch.ones(64, device=device, dtype=torch.bfloat16)

    def f(q, k, pos, gq, gk):
        oq, ok = _ops().qk_norm_rope(q, k, w, w, cos, sin, pos, [8, 24], False, 1e-6)
        return (oq, ok, *_ops().qk_norm_rope_bwd(q, k, w, w, gq, gk, cos, sin, pos, [8, 24], False, 1e-6, True))

    def inputs(seed):
        t = [make(2, h, 19, 64, torch.bfloat16, device, seed + i) for i, h in enumerate((4, 2, 4, 2))]
        return t[0], t[1], make_positions("abs", 2, 2, 19, 64, device, seed), t[2], t[3]

    args = inputs(0)
    want = f(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = f(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    runner = HIPGraphRunner(f)
    runner.capture(*args, clone_args=True)
    for step in range(3):
        args = inputs(10 + step)
        (torch.randn(256, 256, device=device) @ torch.randn(256, 256, device=device)).sum().item()
        got = [t.clone() for t in runner(*args)]
        assert all(torch.equal(a, b) for a, b in zip(f(*args), got))


def test_under_the_compiler(device):
    """The ops inside a compiled function, next to the attention that reads their results."""
    from xpu_graph_amd import mi355x_compiler

    cos, sin = tables(128, 64, device, torch.float32, 3, False)
    w = torch.ones(128, device=device, dtype=torch.bfloat16)
    pos = make_positions("abs", 3, 2, 50, 128, device, 1)

    def f(x):
        heads = x.view(2, 50, 8, 128).transpose(1, 2)
        q, k = torch.ops.xpu_ops.qk_norm_rope(heads[:, :4], heads[:, 4:6], w, w, cos, sin, pos, [16, 24, 24], True, 1e-6)
        return torch.ops.xpu_ops.sdpa(q, k, heads[:, 6:], True, 128**-0.5)

    _ops()
    x = torch.randn(2, 50, 1024, device=device).bfloat16()
    with torch.no_grad():
        assert torch.equal(torch.compile(f, backend=mi355x_compiler(), dynamic=False)(x), f(x))


def test_the_kernels_refuse_what_they_cannot_take(device):
    x = make(1, 2, 4, 64, torch.bfloat16, device, 1)
    cos, sin = tables(4, 32, device, torch.float32, 1, False)
    with pytest.raises(TypeError):
        _ops().rope_axes(x.double(), cos.double(), sin.double(), None, [])
    with pytest.raises(ValueError):
        _ops().rope_axes(x, cos, sin, torch.zeros(4, dtype=torch.int64), [])  # positions on the host
    with pytest.raises(ValueError):
        _ops().qk_norm_rope(x, x[..., :32], None, None, cos, sin, None, [], False, 1e-6)

def test_dimensions_of_one_element_have_no_stride_that_counts(device):
    S, D = 33, 64
    q, k = (torch.randn(S * D, device=device).bfloat16().as_strided((1, 1, S, D), (S * D + 1, S * D + 3, D, 1)) for _ in range(2))
    assert q.is_contiguous() and q.stride(0) % 8
    cos, sin = tables(S, D // 2, device, torch.float32, 1, False)
    w = 1 + 0.1 * torch.randn(D, device=device)
    plain = lambda x: x.reshape(-1).clone().view(x.shape)  # noqa: E731
    assert torch.equal(_ops().rope_axes(q, cos, sin, None, []), _ops().rope_axes(plain(q), cos, sin, None, []))

    def run(q, k):
        return (*_ops().qk_norm_rope(q, k, w, w, cos, sin, None, [], False, 1e-6), *_ops().qk_norm_rope_bwd(q, k, w, w, k, q, cos, sin, None, [], False, 1e-6, True))

    assert all(torch.equal(a, b) for a, b in zip(run(q, k), run(plain(q), plain(k))))
    moved = [torch.empty(x.numel() + 1, dtype=x.dtype, device=device)[1:].view(x.shape).copy_(x) for x in (q, k)]  # off 16 bytes
    assert all(torch.equal(a, b) for a, b in zip(run(*moved), run(plain(q), plain(k))))


def test_gradients_that_do_not_exist_are_refused(device):
    x = make(1, 2, 4, 64, torch.bfloat16, device, 1).requires_grad_()
    cos, sin = tables(4, 32, device, torch.float32, 1, False)
    y = _ops().rope_axes(x, cos, sin, None, [])
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        dx.sum().backward()
    with pytest.raises(NotImplementedError, match="tables"):
        _ops().rope_axes(x, cos.clone().requires_grad_(), sin, None, [])
    with pytest.raises(NotImplementedError, match="tables"):
        _ops().qk_norm_rope(x, x, None, None, cos, sin.clone().requires_grad_(), None, [], False, 1e-6)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        z = x.detach()
        _ops().rope_axes(torch.autograd.forward_ad.make_dual(z, z), cos, sin, None, [])


@pytest.mark.parametrize("layout", ["heads", "tokens", "packed", "batch inside", "shared", "one head", "odd"])
def test_results_lie_as_the_shape_functions_say(device, layout):
    B, H, S, D = 2, 3, 5, 64
    x = {
        "heads": lambda: torch.randn(B, H, S, D),
        "tokens": lambda: torch.randn(B, S, H, D).transpose(1, 2),
        "packed": lambda: torch.randn(B, S, 3 * H * D).view(B, S, 3 * H, D).transpose(1, 2)[:, H : 2 * H],
        "batch inside": lambda: torch.randn(S, B, 2 * H, D).permute(1, 2, 0, 3)[:, :H],
        "shared": lambda: torch.randn(B, 1, S, D).expand(B, H, S, D),
        "one head": lambda: torch.randn(B, S, 1, D).transpose(1, 2),
        "odd": lambda: torch.randn(B, S, H, D + 3).transpose(1, 2)[..., 1 : D + 1],
    }[layout]().bfloat16().to(device)
    cos, sin = tables(S, D // 2, device, torch.float32, 1, False)
    args = lambda x, c, s: (x, x, None, None, c, s, None, [], False, 1e-6)  # noqa: E731
    got = _ops().qk_norm_rope(*args(x, cos, sin))
    as_meta = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="meta")  # noqa: E731
    told = _ops().qk_norm_rope(*args(as_meta(x), as_meta(cos), as_meta(sin)))
    assert [t.stride() for t in got] == [t.stride() for t in told]
    want = _ops().qk_norm_rope(*args(x.contiguous(), cos, sin))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    lin = lambda x, g: _ops().linear_attn(x, x, x, g, None, None, 1.0)  # noqa: E731
    g = torch.zeros(x.shape[1], device=device)
    assert [t.stride() for t in lin(x, g)] == [t.stride() for t in lin(as_meta(x), as_meta(g))]


@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,S", [(0, 2, 1, 5), (2, 2, 1, 0), (2, 0, 0, 5)])
def test_the_entry_point_sums_weight_gradients_over_no_rows(device, w_dtype, B, H, Hkv, S):
    """Weight gradients are sums over rows; over none they are zero, and written."""
    import ctypes

    lib = _xops()._lib.lib()
    D = 64
    cos, sin = tables(8, D // 2, device, torch.float32, 1, False)
    r = _xops()._lib.XgRotary(cos.data_ptr(), sin.data_ptr(), 8, D // 2, D // 2, D)
    r.axes, r.table_dtype = 1, 0
    dtype = torch.bfloat16 if w_dtype == torch.float32 else w_dtype
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    assert lib.xg_qk_norm_rope_bwd_workspace_floats(B, H, Hkv, S, D) == 0
    both = [torch.full((D,), 7.0, device=device, dtype=w_dtype) for _ in range(2)]
    for gws in (both, (both[0], None), (None, None)):
        for x in both:
            x.fill_(7.0)
        p = [x.data_ptr() if x is not None else None for x in gws]
        rc = lib.xg_qk_norm_rope_bwd(*[None] * 8, *p, None, 0, B, H, Hkv, S, D, *[st] * 6, r, 1e-6, code[dtype], code[w_dtype], torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        for x, wanted in zip(both, gws):
            assert (x == (0 if wanted is not None else 7)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("w_types", [(torch.float64, torch.float64), (torch.float64, None), (torch.float16, torch.float64)])
def test_weights_of_other_types_have_gradients_of_their_own_type(device, dtype, w_types):
    """The kernels read such weights as fp32, forward and backward: the gradient is the fp32 one, in the weight's type."""
    q, k = make(2, 4, 19, 64, dtype, device, 1), make(2, 2, 19, 64, dtype, device, 2)
    gq, gk = make(2, 4, 19, 64, dtype, device, 3), make(2, 2, 19, 64, dtype, device, 4)
    ws = [(1 + 0.2 * torch.randn(64, device=device)).to(t).requires_grad_() if t else None for t in w_types]
    wf = [w.detach().float() if w is not None else None for w in ws]
    turn = (*tables(19, 32, device, torch.float32, 1, False), None, [], False, 1e-6)
    out = _ops().qk_norm_rope(q, k, *ws, *turn)
    assert all(torch.equal(a, b) for a, b in zip(out, _ops().qk_norm_rope(q, k, *wf, *turn)))
    want = _ops().qk_norm_rope_bwd(q, k, *wf, gq, gk, *turn, True)
    there = [i for i, w in enumerate(ws) if w is not None]
    got = torch.autograd.grad(out, [ws[i] for i in there], (gq, gk), allow_unused=True)
    for i, gw in zip(there, got):
        assert gw.dtype == ws[i].dtype and torch.equal(gw, want[2 + i].to(gw.dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("case,S", [(CASES[1], 3001), (CASES[4], 2001), (CASES[6], 2001), (CASES[6], 6001)])
def test_two_and_four_heads_a_thread_of_the_other_types(device, dtype, case, S):
    check_qk(device, dtype, case, 2, 9, 3, S, "own")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case,S", [(CASES[6], 1501), (CASES[6], 6001), (CASES[4], 6001), (CASES[2], 9001)])
def test_two_and_eight_heads_a_thread_of_the_other_types(device, dtype, case, S):
    D, R, sections, woven, kind, per, _ = case
    B, H, P = 2, 11, 70
    x = make(B, H + 2, S, D, dtype, device, 5)[:, 1:-1]  # a part of something else
    cos, sin = tables(P if kind != "none" else S, R // 2, device, torch.float32, 2, per == 2)
    pos = make_positions(kind if kind != "s" else "bs", max(len(sections), 1), B, S, P, device, 3)
    ang = angles(cos, sin, pos, sections, woven, B, S, R)
    assert_rounded_once(_ops().rope_axes(x, cos, sin, pos, sections, woven), *turn(x.double(), ang, R), "rope_axes")
    assert_rounded_once(_ops().rope_axes_bwd(x, cos, sin, pos, sections, woven), *turn_back(x.double(), ang, R), "rope_axes_bwd")
