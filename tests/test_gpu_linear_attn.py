"""Linear attention with a decay per head on the GPU (xpu_ops::linear_attn, its gradients, linear_attn_step) against the
definition in 64 bits:

    S_t = lam S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t

Tolerances.  out and the gradients are sums of products a b c (a, c rows, b a score or a state element) rounded once; in front
of that rounding bf16 rounds the scores and the states once (half a step, 2^-8, of each product), fp16 keeps them to 16 bits
(2^-16).  Element by element that gives half a step of the result plus that share of the sum of the products' magnitudes.  The
2-norm is sharper: a rounding error is uniform in half a step, at most 2^-8 / sqrt(3) of its term in the mean square, and the
terms of random inputs add up without direction, so three roundings (score, state, result) give at most 2^-8 of the result's
norm, one of them 2^-11 / sqrt(3) for fp16 (and 2^-16 for the rest).  States are fp32: 24 bits of every product, so an element is
off by 2^-24 of the magnitudes for each of the roundings on its way: the factor, the product, the 64 products of a chunk and one
decay and one addition per chunk and segment.  A decay is exp2(y), y = fl(fl(log_decay log2(e)) n): log2(e) is off by 2^-25 of
itself, and two roundings follow, so y is off by at most 2.5 x 2^-24 of itself, and with x = -log_decay n = -y ln 2 the term it
weighs by 2.5 x 2^-24; exponents of products of decays add up, so x is at most |log_decay| S, and beyond 104 a term is below the
smallest fp32 number."""
import math

import pytest
import torch

from xpu_graph_amd import HIPGraphRunner

pytestmark = pytest.mark.gpu


def _xops():
    import xpu_graph_amd.ops as xops

    return xops


def _ops():
    _xops()
    return torch.ops.xpu_ops


def make(shape, dtype, device, seed, layout="bshd"):
    g = torch.Generator().manual_seed(seed)
    B, H, S, D = shape
    if layout == "bhsd":
        return torch.randn(B, H, S, D, generator=g).to(dtype).to(device)
    return torch.randn(B, S, H, D, generator=g).to(dtype).to(device).transpose(1, 2)


def decays(H, device, kind="mixed"):
    if kind == "mixed":  # from no decay at all to no memory at all
        vals = [0.0, -0.01, -1e-4, -0.2, -1.0, -30.0, float("-inf"), -0.003]
        return torch.tensor([vals[h % len(vals)] for h in range(H)], device=device)
    return -torch.exp2(-1.0 - 9.0 * torch.arange(H, device=device, dtype=torch.float32) / max(H - 1, 1))


def powers(g, n):
    """lam^n in 64 bits, [H, *n.shape]; 0 where n < 0 (and lam^0 = 1 whatever lam)."""
    g = g.double().clamp_min(-1e30)  # minus infinity: 0 from the first power on
    e = g.view(-1, *([1] * n.dim())) * n.double()
    return torch.where(n < 0, torch.zeros_like(e), torch.exp(e))


def reference(q, k, v, g, state, lengths, scale, d_out=None, d_state=None):
    """Values and the magnitudes of what they sum, by name, in 64 bits, from the definition written out over token pairs."""
    B, H, S, D = q.shape
    group = H // k.shape[1]
    dev = q.device
    length = lengths.long().clamp(0, S) if lengths is not None else torch.full((B,), S, device=dev)
    t = torch.arange(S, device=dev)
    alive = (t < length[:, None])[:, None, :, None]
    wide = lambda x: torch.where(alive, x.double().repeat_interleave(H // x.shape[1], 1), 0.0)  # noqa: E731
    q, k, v = wide(q), wide(k), wide(v)
    M = powers(g, t[:, None] - t)  # [H, S, S]
    reach = powers(g, t + 1)[None, :, :, None]
    left = powers(g, length[:, None] - 1 - t).transpose(0, 1)[..., None]  # [B, H, S, 1]
    whole = powers(g, length).transpose(0, 1)[..., None, None]
    s0 = state.double() if state is not None else q.new_zeros(B, H, D, D)
    sc = torch.tensor(float(scale), dtype=torch.float64, device=dev)
    out = {}

    def put(name, f, *args):
        out[name] = (f(*args), f(*(a.abs() for a in args)))

    put("o", lambda q, k, v, s0, sc: sc * (((q @ k.transpose(-1, -2)) * M) @ v + reach * (q @ s0)) * alive, q, k, v, s0, sc)
    put("state", lambda k, v, s0: (k * left).transpose(-1, -2) @ v + whole * s0, k, v, s0)
    if d_out is not None:
        go = wide(d_out)
        ds = d_state.double() if d_state is not None else q.new_zeros(B, H, D, D)
        Mt = M.transpose(-1, -2)
        narrow = lambda x: x.view(B, H // group, group, S, D).sum(2) * alive[:, : H // group]  # noqa: E731
        put("dq", lambda go, v, k, s0, sc: sc * (((go @ v.transpose(-1, -2)) * M) @ k + reach * (go @ s0.transpose(-1, -2))) * alive, go, v, k, s0, sc)
        put("dk", lambda v, go, q, ds, sc: narrow(sc * (((v @ go.transpose(-1, -2)) * Mt) @ q) + left * (v @ ds.transpose(-1, -2))), v, go, q, ds, sc)
        put("dv", lambda k, q, go, ds, sc: narrow(sc * (((k @ q.transpose(-1, -2)) * Mt) @ go) + left * (k @ ds)), k, q, go, ds, sc)
        put("d_state", lambda q, go, ds, sc: sc * ((q * reach).transpose(-1, -2) @ go) + whole * ds, q, go, ds, sc)
    return out


def check(name, got, want, mag, S, g):
    assert torch.isfinite(got).all(), name
    err = (got.double() - want).abs()
    if got.dtype == torch.float32:
        n_chunk = -(-S // 64)
        x = (g.double().abs() * max(S, 1)).clamp_max(104)[:, None, None]
        tol = 2.0**-24 * (6 + min(S, 64) + 3 * n_chunk + 2.5 * x) * mag + 1e-37
        assert (err <= tol).all(), f"{name}: {(err / tol).max().item():.3f} of the tolerance"
        return
    half = torch.finfo(got.dtype).eps / 2
    inner = 2 * 2.0**-8 if got.dtype == torch.bfloat16 else 4 * 2.0**-16
    tol = half * want.abs() + (inner + 2.0**-24 * 200) * mag + torch.finfo(got.dtype).smallest_normal * half
    assert (err <= tol).all(), f"{name}: {(err / tol).max().item():.3f} of the tolerance"
    if want.numel() >= 4096 and want.norm() > 0:
        rel = (err.norm() / want.norm()).item()
        most = 2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-11 / 3**0.5 * 1.1 + 2.0**-14
        assert rel <= most, f"{name}: relative error {rel:.2e}, at most {most:.2e}"


def run_all(device, dtype, B, H, Hkv, S, D, *, state=True, lengths=None, d_state=True, kind="mixed", layout="bshd", seed=1, scale=None, poison=True):
    scale = D**-0.5 if scale is None else scale
    q, k, v = make((B, H, S, D), dtype, device, seed, layout), make((B, Hkv, S, D), dtype, device, seed + 1, layout), make((B, Hkv, S, D), dtype, device, seed + 2, layout)
    go = make((B, H, S, D), dtype, device, seed + 3, layout)
    g = decays(H, device, kind)
    gen = torch.Generator().manual_seed(seed + 4)
    s0 = torch.randn(B, H, D, D, generator=gen).to(device) if state else None
    ds = torch.randn(B, H, D, D, generator=gen).to(device) if d_state else None
    n = torch.tensor(lengths, device=device) if lengths is not None else None
    want = reference(q, k, v, g, s0, n, scale, go, ds)
    if n is not None and poison:  # what lies behind a sequence is not read
        for i, bad in zip(range(B), (float("nan"), float("inf"), float("-inf"), 1e4)):
            for x in (q, k, v, go):
                x[i, :, max(0, min(S, lengths[i])) :] = bad
    o, s = _ops().linear_attn(q, k, v, g, s0, n, scale)
    assert o.shape == q.shape and o.dtype == dtype and o.stride() == q.stride()
    check("o", o, *want["o"], S, g)
    check("state", s, *want["state"], S, g)
    dq, dk, dv, d0 = _ops().linear_attn_bwd(q, k, v, g, s0, n, go, ds, scale, True)
    for name, x, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        assert x.shape == like.shape and x.dtype == dtype and x.stride() == like.stride()
        check(name, x, *want[name], S, g)
    check("d_state", d0, *want["d_state"], S, g)


LENGTHS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 191, 256, 700]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", LENGTHS)
def test_lengths(device, dtype, D, S):
    run_all(device, dtype, 1, 8, 8, S, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("state,d_state", [(False, False), (True, False), (False, True)])
def test_without_states(device, dtype, D, state, d_state):
    run_all(device, dtype, 2, 3, 3, 150, D, state=state, d_state=d_state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,S,D", [(1, 6, 2, 70, 64), (2, 8, 1, 333, 128), (1, 12, 4, 129, 128), (3, 2, 1, 1, 64), (4, 4, 2, 333, 64), (2, 16, 4, 70, 128), (2, 16, 4, 700, 128)])
def test_shared_heads(device, dtype, B, H, Hkv, S, D):
    run_all(device, dtype, B, H, Hkv, S, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,lengths", [(1, [0, 1, 1, 0]), (64, [64, 63, 1, 0]), (200, [0, 200, 65, 128]), (449, [1, 449, 448, 64]), (100, [-3, 1000, 64, 50])])
def test_ragged_batches_do_not_read_what_lies_behind(device, dtype, S, lengths):
    run_all(device, dtype, 4, 4, 2, S, 64, lengths=lengths)
    run_all(device, dtype, 4, 2, 2, S, 128, lengths=lengths)


@pytest.mark.parametrize("B,H,S,D", [(4, 128, 130, 64), (8, 80, 100, 128), (2, 300, 64, 64)])
def test_many_heads_run_as_one_segment(device, B, H, S, D):
    assert _xops()._lib.lib().xg_linear_attn_workspace_floats(B, H, S, D) == 0
    run_all(device, torch.bfloat16, B, H, H, S, D, kind="model")


def test_few_heads_are_cut_into_segments(device):
    assert _xops()._lib.lib().xg_linear_attn_workspace_floats(1, 2, 2000, 64) > 0
    run_all(device, torch.bfloat16, 1, 2, 2, 2000, 64, kind="model")
    run_all(device, torch.float16, 2, 2, 1, 1999, 128, kind="model", lengths=[700, 1999])


def test_a_long_sequence_keeps_its_state(device):
    """16384 tokens against a token by token evaluation in 64 bits of the final state, with a memory of all of them."""
    S, D, H = 16384, 64, 3
    q, k, v = (make((1, H, S, D), torch.bfloat16, device, i) for i in range(3))
    g = torch.tensor([0.0, -1e-4, -0.02], device=device)
    _, s = _ops().linear_attn(q, k, v, g, None, None, 0.125)
    w = powers(g, S - 1 - torch.arange(S, device=device))[None, :, :, None]
    want = (k.double() * w).transpose(-1, -2) @ v.double()
    mag = (k.double().abs() * w).transpose(-1, -2) @ v.double().abs()
    check("state", s, want, mag, S, g)


@pytest.mark.parametrize("layout", ["bhsd", "packed", "shared", "odd"])
def test_layouts(device, layout):
    B, H, S, D = 2, 4, 130, 64
    if layout == "packed":
        heads = make((B, 3 * H, S, D), torch.bfloat16, device, 1)
        q, k, v = heads[:, :H], heads[:, H : 2 * H], heads[:, 2 * H :]
    elif layout == "shared":  # one key head seen by all, a broadcast view
        q, k, v = make((B, H, S, D), torch.bfloat16, device, 1), *(make((B, 1, S, D), torch.bfloat16, device, i).expand(B, H, S, D) for i in (2, 3))
    elif layout == "odd":  # a pitch and a start that are no multiples of 16 bytes
        q, k, v = (torch.randn(B, H, S, D + 3, device=device).bfloat16()[..., 1 : D + 1] for _ in range(3))
    else:
        q, k, v = (make((B, H, S, D), torch.bfloat16, device, i, "bhsd") for i in range(3))
    g, go = decays(H, device), make((B, H, S, D), torch.bfloat16, device, 9)
    got = (*_ops().linear_attn(q, k, v, g, None, None, 0.1), *_ops().linear_attn_bwd(q, k, v, g, None, None, go, None, 0.1, False))
    q, k, v = (x.contiguous() for x in (q, k, v))
    want = (*_ops().linear_attn(q, k, v, g, None, None, 0.1), *_ops().linear_attn_bwd(q, k, v, g, None, None, go, None, 0.1, False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scales_and_values_at_the_ends_of_the_types(device):
    run_all(device, torch.bfloat16, 1, 4, 4, 100, 64, scale=-0.3)
    run_all(device, torch.float16, 1, 4, 4, 100, 64, scale=1.0)
    # fp16: states and scores far beyond its range, results inside it
    B, H, S, D = 1, 2, 300, 64
    q, k, v = (make((B, H, S, D), torch.float16, device, i) for i in range(3))
    q, k, v, g = q * 0.001, k * 200, (v.abs() + 1) * 100, decays(H, device)
    want = reference(q, k, v, g, None, None, 0.05)
    assert want["state"][0].abs().max() > 1e6 and want["o"][0].abs().max() < 6e4
    o, s = _ops().linear_attn(q, k, v, g, None, None, 0.05)
    check("o", o, *want["o"], S, g)
    check("state", s, *want["state"], S, g)
    # ... and the small ones
    q, k, v = q * 1000, k * 2.0**-20, v * 2.0**-16
    want = reference(q, k, v, g, None, None, 1.0)
    o, s = _ops().linear_attn(q, k, v, g, None, None, 1.0)
    check("state", s, *want["state"], S, g)


def test_a_prompt_in_pieces_and_token_by_token_equals_the_whole(device):
    """The states handed over are fp32 results, so pieces, steps and the whole agree to the tolerances of one call."""
    for dtype, D, Hkv in ((torch.bfloat16, 128, 4), (torch.float16, 64, 2)):
        B, H, S, cut = 2, 4, 173, 90
        q, k, v = make((B, H, S, D), dtype, device, 1), make((B, Hkv, S, D), dtype, device, 2), make((B, Hkv, S, D), dtype, device, 3)
        g, scale = decays(H, device), D**-0.5
        want = reference(q, k, v, g, None, None, scale)
        o1, s1 = _ops().linear_attn(q[:, :, :cut], k[:, :, :cut], v[:, :, :cut], g, None, None, scale)
        o2, s2 = _ops().linear_attn(q[:, :, cut:], k[:, :, cut:], v[:, :, cut:], g, s1, None, scale)
        check("o", torch.cat([o1, o2], 2), *want["o"], S, g)
        check("state", s2, *want["state"], S, g)
        st, rows = s1.clone(), []
        for t in range(cut, S):
            rows.append(_ops().linear_attn_step(q[:, :, t : t + 1], k[:, :, t : t + 1], v[:, :, t : t + 1], g, st, scale))
        check("o by steps", torch.cat(rows, 2), want["o"][0][:, :, cut:], want["o"][1][:, :, cut:], S, g)
        check("state by steps", st, *want["state"], 64 * S, g)  # a decay and an addition per token


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,D", [(1, 1, 1, 64), (3, 6, 2, 128), (5, 4, 4, 64), (64, 8, 1, 128)])
def test_step(device, dtype, B, H, Hkv, D):
    q, k, v = make((B, H, 1, D), dtype, device, 1), make((B, Hkv, 1, D), dtype, device, 2), make((B, Hkv, 1, D), dtype, device, 3)
    g = decays(H, device)
    pool = torch.randn(B + 2, H + 1, D, D, device=device)  # states inside a larger tensor
    before = pool.clone()
    state = pool[1 : B + 1, :H]
    want = reference(q, k, v, g, state.clone(), None, 0.2)
    o = _ops().linear_attn_step(q, k, v, g, state, 0.2)
    assert o.shape == q.shape and o.dtype == dtype
    check("o", o, *want["o"], 1, g)
    check("state", state, *want["state"], 1, g)
    pool[1 : B + 1, :H] = before[1 : B + 1, :H]
    assert torch.equal(pool, before)  # nothing around them was touched


def test_step_reads_any_alignment(device):
    B, H, D = 2, 3, 64
    base = torch.randn(B, H, 3 * D + 7, device=device).bfloat16()
    q, k, v = (base[:, :, None, 1 + i * (D + 1) : 1 + i * (D + 1) + D] for i in range(3))
    g = decays(H, device)
    a, b = torch.zeros(B, H, D, D, device=device), torch.zeros(B, H, D, D, device=device)
    assert torch.equal(_ops().linear_attn_step(q, k, v, g, a, 1.0), _ops().linear_attn_step(*(x.contiguous() for x in (q, k, v)), g, b, 1.0))
    assert torch.equal(a, b)


def test_empty_inputs(device):
    g = decays(2, device)
    s0 = torch.randn(1, 2, 64, 64, device=device)
    e = torch.empty(1, 2, 0, 64, device=device, dtype=torch.bfloat16)
    o, s = _ops().linear_attn(e, e, e, g, s0, None, 1.0)
    assert o.shape == e.shape and torch.equal(s, s0)
    assert (_ops().linear_attn(e, e, e, g, None, None, 1.0)[1] == 0).all()
    dq, dk, dv, d0 = _ops().linear_attn_bwd(e, e, e, g, s0, None, e, s0, 1.0, True)
    assert dq.shape == e.shape and torch.equal(d0, s0)
    n = torch.empty(0, 2, 5, 64, device=device, dtype=torch.bfloat16)
    assert _ops().linear_attn(n, n, n, g, None, None, 1.0)[1].shape == (0, 2, 64, 64)
    n = n[:, :, :1]
    assert _ops().linear_attn_step(n, n, n, g, torch.empty(0, 2, 64, 64, device=device), 1.0).shape == n.shape


def test_gradients_through_autograd_and_against_differences(device):
    """The result is linear in q, in k, in v and in the state, one at a time, so a central difference of any step is the
    derivative, up to the roundings of the two results; the inputs are small whole numbers, exact in bf16."""
    _xops().enable_autograd()
    B, H, Hkv, S, D, scale = 1, 4, 2, 75, 64, 0.125
    gen = torch.Generator().manual_seed(5)
    whole = lambda *s: torch.randint(-3, 4, s, generator=gen).to(device)  # noqa: E731
    leaves = [whole(B, H, S, D).bfloat16(), whole(B, Hkv, S, D).bfloat16(), whole(B, Hkv, S, D).bfloat16(), whole(B, H, D, D).float()]
    leaves = [t.requires_grad_() for t in leaves]
    g = torch.tensor([0.0, -0.05, -0.5, -3.0], device=device)
    up_o, up_s = whole(B, H, S, D).bfloat16(), whole(B, H, D, D).float()

    def forward(q, k, v, s0):
        return _ops().linear_attn(q, k, v, g, s0, None, scale)

    grads = torch.autograd.grad(forward(*leaves), leaves, (up_o, up_s))
    for i, leaf in enumerate(leaves):
        d = whole(*leaf.shape).to(leaf.dtype)
        both, noise = [], 0.0
        for sign in (1, -1):
            o, s = forward(*(t.detach() + (sign * d if j == i else 0) for j, t in enumerate(leaves)))
            both.append((o.double() * up_o.double()).sum() + (s.double() * up_s.double()).sum())
            noise += (o.double() * up_o.double()).norm().item() * 2.0**-8 + (s.double() * up_s.double()).norm().item() * 2.0**-20
        slope = ((both[0] - both[1]) / 2).item()
        want = (grads[i].double() * d.double()).sum().item()
        # independent errors of at most 2^-8 a term in the mean square, on both sides: four of their norm
        noise = 4 * (noise / 2 + (grads[i].double() * d.double()).norm().item() * 2.0**-8)
        assert abs(slope - want) <= noise, (i, slope, want, noise)
    q = leaves[0]
    o, s = forward(*leaves)
    (only,) = torch.autograd.grad(s, leaves[1], up_s, retain_graph=True)  # the gradient of the state alone
    want = _ops().linear_attn_bwd(*leaves[:3], g, leaves[3], None, torch.zeros_like(q), up_s, scale, False)[1]
    assert torch.equal(only, want)
    (only,) = torch.autograd.grad(o, q, up_o)
    assert torch.equal(only, _ops().linear_attn_bwd(*leaves[:3], g, leaves[3], None, up_o, None, scale, False)[0])
    with pytest.raises(NotImplementedError):
        _ops().linear_attn(q, leaves[1], leaves[2], g.clone().requires_grad_(), None, None, scale)[0].sum().backward()


def test_results_do_not_depend_on_the_run(device):
    first = None
    for _ in range(3):
        q, k, v, go = (make((1, h, 900, 64), torch.bfloat16, device, i) for i, h in enumerate((6, 2, 2, 6)))
        out = (*_ops().linear_attn(q, k, v, decays(6, device), None, None, 0.1), *_ops().linear_attn_bwd(q, k, v, decays(6, device), None, None, go, None, 0.1, True))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_side_stream_and_graph_replays(device):
    g = decays(6, device)

    def f(q, k, v, go, s0, n):
        o, s = _ops().linear_attn(q, k, v, g, s0, n, 0.1)
        grads = _ops().linear_attn_bwd(q, k, v, g, s0, n, go, s, 0.1, True)
        st = s.clone()
        row = _ops().linear_attn_step(q[:, :, :1], k[:, :, :1], v[:, :, :1], g, st, 0.1)
        return (o, s, *grads, row, st)

    def inputs(seed):
        t = [make((2, h, 600, 64), torch.bfloat16, device, seed + i) for i, h in enumerate((6, 2, 2, 6))]
        return (*t, torch.randn(2, 6, 64, 64, device=device), torch.tensor([600 - seed, 300 + seed], device=device))

    args = inputs(0)
    want = f(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = f(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    runners = [HIPGraphRunner(f) for _ in range(2)]  # two recordings, each with workspaces of its own
    for r in runners:
        r.capture(*args, clone_args=True)
    for step in range(3):
        args = inputs(10 + step)
        (torch.randn(256, 256, device=device) @ torch.randn(256, 256, device=device)).sum().item()
        for r in runners:
            got = [t.clone() for t in r(*args)]
            assert all(torch.equal(a, b) for a, b in zip(f(*args), got))


def layer(x, w_in, w_out, wq, wk, cos, sin, positions, g, state, H, D):
    """One attention layer as a model has it: projection, norm and rotation, linear attention, projection."""
    B, S, _ = x.shape
    heads = torch.nn.functional.linear(x, w_in).view(B, S, 3 * H, D).transpose(1, 2)
    q, k = torch.ops.xpu_ops.qk_norm_rope(heads[:, :H], heads[:, H : 2 * H], wq, wk, cos, sin, positions, [], False, 1e-6)
    if S == 1:
        o = torch.ops.xpu_ops.linear_attn_step(q, k, heads[:, 2 * H :], g, state, D**-0.5)
    else:
        o, state = torch.ops.xpu_ops.linear_attn(q, k, heads[:, 2 * H :], g, state, None, D**-0.5)
    return torch.nn.functional.linear(o.transpose(1, 2).reshape(B, S, H * D), w_out), state


def test_a_layer_prompts_and_decodes(device):
    """Prompt, then tokens: compiled and plain, against the layer in fp32 over the whole sequence."""
    from xpu_graph_amd import mi355x_compiler

    _ops()
    B, S, cut, H, D, E = 2, 90, 83, 4, 64, 128
    bf = torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    mk = lambda *s, m=1.0: (torch.randn(*s, generator=gen) * m).to(bf).to(device)  # noqa: E731
    x, w_in, w_out = mk(B, S, E), mk(3 * H * D, E, m=E**-0.5), mk(E, H * D, m=(H * D) ** -0.5)
    wq, wk = 1 + mk(D, m=0.1), 1 + mk(D, m=0.1)
    angle = torch.arange(S, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    cos, sin = angle.cos().float().to(device), angle.sin().float().to(device)
    g = decays(H, device, "model")
    pos = torch.arange(S, device=device)

    def run(fn):
        with torch.no_grad():
            y, state = fn(x[:, :cut], w_in, w_out, wq, wk, cos, sin, pos[:cut], g, None, H, D)
            rows = [y]
            for t in range(cut, S):
                rows.append(fn(x[:, t : t + 1], w_in, w_out, wq, wk, cos, sin, pos[t : t + 1], g, state, H, D)[0])
        return torch.cat(rows, 1), state

    y, state = run(layer)
    yc, sc = run(torch.compile(layer, backend=mi355x_compiler(), dynamic=False))

    xf = x.double()
    heads = (xf @ w_in.double().T).view(B, S, 3 * H, D).transpose(1, 2)

    def turned(h, w):
        n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        a, b = n[..., : D // 2], n[..., D // 2 :]
        c, s = cos.double(), sin.double()
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    ref = reference(turned(heads[:, :H], wq), turned(heads[:, H : 2 * H], wk), heads[:, 2 * H :], g, None, None, D**-0.5)
    want = ref["o"][0].transpose(1, 2).reshape(B, S, H * D) @ w_out.double().T
    # roundings in the chain: the projection, the turned q and k (two factors), the attention and its two inner ones, the last
    # projection; 2^-8 / sqrt(3) each in the mean square, v's among them
    for got, st in ((y, state), (yc, sc)):
        assert ((got.double() - want).norm() / want.norm()).item() <= 2.0**-8 / 3**0.5 * 8**0.5
        assert ((st.double() - ref["state"][0]).norm() / ref["state"][0].norm()).item() <= 2.0**-8 / 3**0.5 * 4**0.5


def test_a_training_step_of_the_layer(device):
    _xops().enable_autograd()
    B, S, H, D, E = 2, 100, 2, 64, 64
    bf = torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    mk = lambda *s, m=1.0: (torch.randn(*s, generator=gen) * m).to(bf).to(device)  # noqa: E731
    x = mk(B, S, E)
    leaves = [mk(3 * H * D, E, m=E**-0.5), mk(E, H * D, m=(H * D) ** -0.5), 1 + mk(D, m=0.1), 1 + mk(D, m=0.1)]
    leaves = [t.requires_grad_() for t in leaves]
    ang = torch.rand(S, D // 2, generator=gen) * 6
    cos, sin, g = ang.cos().to(device), ang.sin().to(device), decays(H, device, "model")
    y, _ = layer(x, *leaves, cos, sin, None, g, None, H, D)
    grads = torch.autograd.grad(y, leaves, mk(B, S, E))
    assert all(gr.shape == t.shape and torch.isfinite(gr).all() and gr.abs().max() > 0 for gr, t in zip(grads, leaves))


def test_refusals(device):
    q = make((1, 2, 8, 64), torch.bfloat16, device, 1)
    g = decays(2, device)
    with pytest.raises(ValueError):
        _ops().linear_attn(q, q, q, g.cpu(), None, None, 1.0)  # another device
    with pytest.raises(RuntimeError, match="xg_linear_attn"):
        _ops().linear_attn(q, q, q, g, None, None, math.nan)
    t = q[:, :, :1]
    with pytest.raises(RuntimeError, match="xg_linear_attn"):  # one state seen twice
        _ops().linear_attn_step(t, t, t, g, torch.zeros(1, 1, 64, 64, device=device).expand(1, 2, 64, 64), 1.0)
    with pytest.raises(ValueError):  # a state that could not be updated in place
        _ops().linear_attn_step(t, t, t, g, torch.zeros(1, 2, 64, 64, device=device).transpose(2, 3), 1.0)

def test_dimensions_of_one_element_have_no_stride_that_counts(device):
    """Contiguous to torch, with strides of no whole 16 bytes where a dimension has one element."""
    S, D = 70, 64
    odd = lambda x: x.as_strided(x.shape, (x[0].numel() + 1, x[0, 0].numel() + 3, D, 1))  # noqa: E731
    q, k, v, go = (odd(torch.randn(1, 1, S, D, device=device).bfloat16() * 0.3) for _ in range(4))
    assert q.is_contiguous() and q.stride(0) % 8
    g, s0 = decays(1, device), odd(torch.randn(1, 1, D, D, device=device))
    run = lambda *a: (*_ops().linear_attn(*a[:3], g, a[4], None, 0.1), *_ops().linear_attn_bwd(*a[:3], g, a[4], None, a[3], a[4], 0.1, True))  # noqa: E731
    args = (q, k, v, go, s0)
    assert all(torch.equal(a, b) for a, b in zip(run(*args), run(*(x.reshape(-1).clone().view(x.shape) for x in args))))
    t = (q[:, :, :1], k[:, :, :1], v[:, :, :1])
    plain = s0.reshape(-1).clone().view(s0.shape)
    st = odd(plain.clone())
    assert torch.equal(_ops().linear_attn_step(*t, g, st, 0.1), _ops().linear_attn_step(*t, g, plain, 0.1)) and torch.equal(st, plain)
    # one token, tokens of a huge pitch: nothing is copied or refused, nor is there a second token to reach
    far = torch.as_strided(q.reshape(-1)[:D].clone(), (1, 1, 1, D), (1 << 40, 1 << 40, 1 << 40, 1))
    assert torch.equal(_ops().linear_attn(far, far, far, g, None, None, 0.1)[0], _ops().linear_attn(*[q[:, :, :1]] * 3, g, None, None, 0.1)[0])


def test_starts_off_16_bytes_are_copied(device):
    B, H, S, D = 1, 2, 40, 64
    args = [make((B, H, S, D), torch.bfloat16, device, i, "bhsd") for i in range(4)]
    moved = []
    for x in args:
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=device)[1:].view(x.shape)
        moved.append(y.copy_(x))
    g = decays(H, device)
    s0 = torch.empty(B * H * D * D + 1, device=device)[1:].view(B, H, D, D).normal_()
    run = lambda a, s: (*_ops().linear_attn(*a[:3], g, s, None, 0.1), *_ops().linear_attn_bwd(*a[:3], g, s, None, a[3], s, 0.1, True))  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(run(moved, s0), run(args, s0.clone())))
    with pytest.raises(RuntimeError, match="xg_linear_attn_step"):  # a state is written where it lies
        _ops().linear_attn_step(*(x[:, :, :1] for x in args[:3]), g, s0, 0.1)


def test_a_training_pass_recorded_in_a_graph(device):
    """Forward and backward through autograd in one recording, replayed on new values."""
    B, H, S, D = 2, 2, 200, 64
    g = decays(H, device)
    static = [make((B, H, S, D), torch.bfloat16, device, i).requires_grad_() for i in range(3)]
    s0, go = torch.randn(B, H, D, D, device=device).requires_grad_(), make((B, H, S, D), torch.bfloat16, device, 7)

    def f():
        o, s = _ops().linear_attn(*static, g, s0, None, 0.1)
        grads = torch.autograd.grad((o, s), (*static, s0), (go, s.detach()))
        return (o.detach(), s.detach(), *grads)  # (no graph of these leaves outlives a call)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f()
    for step in range(3):
        with torch.no_grad():
            for i, x in enumerate(static):
                x.copy_(make((B, H, S, D), torch.bfloat16, device, 100 * (step + 1) + i))
            s0.normal_()
        graph.replay()
        seen = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(f(), seen))


def test_gradients_that_do_not_exist_are_refused(device):
    g = decays(2, device)
    q, k, v = (make((1, 2, 8, 64), torch.bfloat16, device, i).requires_grad_() for i in range(3))
    o, _ = _ops().linear_attn(q, k, v, g, None, None, 0.1)
    (dq,) = torch.autograd.grad(o, q, torch.ones_like(o).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):  # a gradient of a gradient
        torch.autograd.grad(dq.sum(), k)
    with pytest.raises(NotImplementedError, match="log_decay"):
        _ops().linear_attn(q, k, v, g.clone().requires_grad_(), None, None, 0.1)
    s0 = torch.zeros(1, 2, 64, 64, device=device)
    with pytest.raises(NotImplementedError, match="linear_attn_step"):
        _ops().linear_attn_step(q[:, :, :1], k[:, :, :1], v[:, :, :1], g, s0, 0.1)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        x = q.detach()
        _ops().linear_attn(torch.autograd.forward_ad.make_dual(x, x), x, x, g, None, None, 0.1)
    # a graph that needs the old state sees that a step has overwritten it
    o, _ = _ops().linear_attn(q, k, v, g, s0, None, 0.1)
    x = q.detach()[:, :, :1]
    _ops().linear_attn_step(x, x, x, g, s0, 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():  # tensors without a version counter
        s1 = torch.zeros(1, 2, 64, 64, device=device)
        y = x.clone()
        assert torch.equal(_ops().linear_attn_step(y, y, y, g, s1, 0.1), _ops().linear_attn_step(x, x, x, g, torch.zeros_like(s1), 0.1))


def test_calls_that_overlap_on_two_streams(device):
    """Workspaces, partial sums and states of one call are not those of another."""
    g = decays(4, device)
    sets = [[make((2, h, 900, 128), torch.bfloat16, device, 10 * i + j) for j, h in enumerate((4, 2, 2, 4))] for i in range(2)]

    def f(q, k, v, go):
        o, s = _ops().linear_attn(q, k, v, g, None, None, 0.1)
        return (o, s, *_ops().linear_attn_bwd(q, k, v, g, None, None, go, s, 0.1, True))

    want = [f(*x) for x in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(f(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(want[i], run))


def entry(name, *args):
    """A C entry point on the current stream; tensors by their addresses, tuples as strides."""
    import ctypes

    lib = _xops()._lib.lib()
    raw = [a.data_ptr() if isinstance(a, torch.Tensor) else (ctypes.c_int64 * len(a))(*a) if isinstance(a, tuple) else a for a in args]
    return getattr(lib, name)(*raw, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("given", [True, False])
def test_entry_points_without_tokens_carry_the_state(device, D, given):
    """S = 0: the state after the last token is the one before the first, the gradient of the initial state that of the final one."""
    B, H, Hkv = 3, 4, 2
    before = torch.randn(B, H, D, D, device=device) if given else None
    want = before if given else torch.zeros(B, H, D, D, device=device)
    st = (0, 0, 0)

    def fwd(out):
        return entry("xg_linear_attn", None, None, None, None, before, None, 0, None, out, None, 0, B, H, Hkv, 0, D, st, st, st, st, 1.0, 2)

    def bwd(out):
        return entry("xg_linear_attn_bwd", *[None] * 6, 0, None, before, None, None, None, out, None, 0, B, H, Hkv, 0, D, *[st] * 7, 1.0, 2)

    for call in (fwd, bwd):
        out = torch.full((B, H, D, D), 7.0, device=device)
        assert call(out) == 0 and torch.equal(out, want)
        assert call(None) == 0
        if given:  # in place
            assert call(before) == 0 and torch.equal(before, want)
        off = torch.full((B * H * D * D + 1,), 7.0, device=device)[1:]
        assert call(off) == -3 and (off == 7).all()


def test_an_empty_prompt_piece_recorded_in_a_graph(device):
    B, H, D = 2, 3, 64
    s0, out, st = torch.randn(B, H, D, D, device=device), torch.zeros(B, H, D, D, device=device), (0, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rc = entry("xg_linear_attn", None, None, None, None, s0, None, 0, None, out, None, 0, B, H, H, 0, D, st, st, st, st, 1.0, 2)
    assert rc == 0
    for _ in range(3):
        s0.normal_()
        out.zero_()
        graph.replay()
        assert torch.equal(out, s0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_key_heads_without_query_heads_get_zero_gradients(device, dtype):
    """A gradient of a key head is a sum over its query heads; over none it is zero."""
    B, Hkv, S, D = 2, 3, 37, 64
    q, g = torch.empty(B, 0, S, D, device=device, dtype=dtype), torch.empty(0, device=device)
    heads = make((B, 2 * Hkv, S, D), dtype, device, 1)
    k, v = heads[:, :Hkv], heads[:, Hkv:]
    s0 = torch.empty(B, 0, D, D, device=device)
    for _ in range(2):
        del_me = [torch.full_like(k, 7.0) for _ in range(4)]  # what the allocator hands out next is not zero
        del del_me
        o, s = _ops().linear_attn(q, k, v, g, s0, None, 1.0)
        dq, dk, dv, d0 = _ops().linear_attn_bwd(q, k, v, g, s0, None, q, s0, 1.0, True)
        assert o.shape == dq.shape == q.shape and s.shape == d0.shape == s0.shape
        assert dk.shape == dv.shape == k.shape and (dk == 0).all() and (dv == 0).all()
    # the entry point writes the rows of its operands and nothing between them
    dk, dv = (torch.full((B, S, Hkv + 1, D), 7.0, device=device, dtype=dtype).transpose(1, 2) for _ in range(2))
    st, code = tuple(dk.stride()[:3]), 2 if dtype == torch.bfloat16 else 1
    n = (0, 0, 0)

    def bwd(dk, dv, Hkv=Hkv):
        return entry("xg_linear_attn_bwd", *[None] * 6, 0, None, None, None, dk, dv, None, None, 0, B, 0, Hkv, S, D, *[n] * 5, st, st, 1.0, code)

    assert bwd(dk, None) == -4 and bwd(dk, None, Hkv=0) == 0 and (dk == 7).all()
    assert bwd(dk, dv) == 0
    for x in (dk, dv):
        assert (x[:, :Hkv] == 0).all() and (x[:, Hkv:] == 7).all()


@pytest.mark.parametrize("B,H,S", [(1, 3, 40), (1, 3, 700), (2, 64, 300)])
def test_the_state_of_the_entry_point_in_place(device, B, H, S):
    """state_out may be state: uncut heads, segments, and an entry of no tokens."""
    D = 64
    lib = _xops()._lib.lib()
    q, k, v = (make((B, H, S, D), torch.bfloat16, device, i, "bhsd") for i in range(3))
    g, s0 = decays(H, device, "model"), torch.randn(B, H, D, D, device=device)
    st, n = tuple(q.stride()[:3]), lib.xg_linear_attn_workspace_floats(B, H, S, D)
    ws = torch.empty(max(n, 1), device=device)
    for lengths in (None, torch.full((B,), S // 2, device=device), torch.zeros(B, dtype=torch.long, device=device)):
        want = _ops().linear_attn(q, k, v, g, s0, lengths, 0.1)
        out, state = torch.empty_like(q), s0.clone()
        assert entry("xg_linear_attn", q, k, v, g, state, lengths, 1, out, state, ws, n, B, H, H, S, D, st, st, st, st, 0.1, 2) == 0
        assert torch.equal(out, want[0]) and torch.equal(state, want[1])


# what one bad element at token j of an operand reaches: its own row ("row"), the rows of the tokens from j on or up to j, whole
# ("rows") or in its own column ("col"); of a state its row or column
REACH = {
    "q": {"o": "row", "dk": "col up to", "dv": "rows up to", "d_state": "row"},
    "k": {"o": "rows from", "state": "row", "dq": "col from", "dv": "row"},
    "v": {"o": "col from", "state": "col", "dq": "rows from", "dk": "row"},
    "go": {"dq": "row", "dk": "rows up to", "dv": "col up to", "d_state": "col"},
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,D,j", [(75, 64, 5), (75, 128, 40), (75, 64, 74), (64, 128, 63), (1, 64, 0), (700, 64, 300), (700, 128, 681)])
@pytest.mark.parametrize("what", list(REACH))
def test_a_bad_token_reaches_only_what_depends_on_it(device, dtype, S, D, j, what):
    """The recurrence is causal: a NaN or an infinity at token j leaves the outputs of earlier tokens (the gradients of later ones)
    and of other columns, heads and batch entries as they are without it."""
    B, H, Hkv, scale = 2, 4, 2, 0.1
    group = H // Hkv
    g = torch.tensor([-0.01, 0.0, -0.2, -0.003], device=device)
    clean = {n: make((B, h, S, D), dtype, device, 1 + i) for i, (n, h) in enumerate((("q", H), ("k", Hkv), ("v", Hkv), ("go", H)))}
    gen = torch.Generator().manual_seed(9)
    s0, ds = (torch.randn(B, H, D, D, generator=gen).to(device) for _ in range(2))
    b, head, col = 1, (2 if what in ("q", "go") else 1), 11
    clean[what][b, head, j, col] = 0.0
    want = reference(clean["q"], clean["k"], clean["v"], g, s0, None, scale, clean["go"], ds)
    hk = head // group if what in ("q", "go") else head
    heads = [head] if what in ("q", "go") else list(range(hk * group, hk * group + group))  # the query heads that it meets
    t = torch.arange(S, device=device)
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = {n: y.clone() for n, y in clean.items()}
        x[what][b, head, j, col] = bad
        o, s = _ops().linear_attn(x["q"], x["k"], x["v"], g, s0, None, scale)
        dq, dk, dv, d0 = _ops().linear_attn_bwd(x["q"], x["k"], x["v"], g, s0, None, x["go"], ds, scale, True)
        for name, got in (("o", o), ("state", s), ("dq", dq), ("dk", dk), ("dv", dv), ("d_state", d0)):
            hurt = torch.zeros(got.shape, dtype=torch.bool, device=device)
            how = REACH[what].get(name)
            if how is not None:
                where = [hk] if name in ("dk", "dv") else heads
                if name in ("state", "d_state"):
                    at = (col, slice(None)) if how == "row" else (slice(None), col)
                    hurt[b, where, at[0], at[1]] = True
                else:
                    rows = t == j if how == "row" else (t >= j if how.endswith("from") else t <= j)
                    cols = torch.arange(D, device=device) == col if how.startswith("col") else torch.ones(D, dtype=torch.bool, device=device)
                    hurt[b, where] = rows[:, None] & cols
            label = f"{name} with {bad} in {what}"
            assert not torch.isfinite(got[hurt]).any(), label
            check(label, torch.where(hurt, want[name][0].to(got.dtype), got), *want[name], S, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,D", [(64, 8, 2, 64), (33, 8, 8, 64), (16, 9, 3, 128)])
def test_step_of_many_heads(device, dtype, B, H, Hkv, D):
    """64 columns a workgroup: from 256 workgroups on."""
    test_step(device, dtype, B, H, Hkv, D)


def state_tolerance(S, D, heads, dtype, x):
    """What a state is off by, relative to the magnitudes that it sums; 2^-24 is half a step of fp32, what a rounding is off by at most.
    On the way of a product into it: its weight, a power (one step: 2) and a scale (1), and 2.5 x for its exponent; the weighed value
    (1), what its three 8-bit parts leave out (1) and the 16 products that one matrix instruction adds (16).  Then, with everything
    added so far, each chunk of 32: the accumulations of its two k-steps (three products of parts each, five of fp16's two-part keys),
    one decay (1) and that power's own error (2).  Each segment: one decay (1), its power (2), one addition (1)."""
    chunks = -(-S // 32)
    segments = max(_xops()._lib.lib().xg_linear_attn_workspace_floats(1, heads, S, D) // (heads * D * D), 1)
    accumulations = 6 if dtype == torch.bfloat16 else 10
    return 2.0**-24 * (5 + 16 + (accumulations + 3) * chunks + 4 * segments + 2.5 * x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,D,H", [(1, 64, 3), (33, 128, 3), (64, 64, 2), (700, 128, 3), (4096, 64, 3), (5000, 128, 160)])
def test_states_to_the_bound_of_chunks_of_32(device, dtype, S, D, H):
    """The final state, token by token in 64 bits, against the bound for the chunks and segments that the kernels use."""
    k, v = (make((1, H, S, D), dtype, device, i) for i in range(2))
    g = torch.tensor([(0.0, -1e-4, -0.02)[h % 3] for h in range(H)], device=device)
    _, s = _ops().linear_attn(k, k, v, g, None, None, 0.125)
    for h in range(0, H, max(1, H // 6)):
        w = powers(g[h : h + 1], S - 1 - torch.arange(S, device=device))[0][:, None]
        kd, vd = k[0, h].double(), v[0, h].double()
        want, mag = (kd * w).T @ vd, (kd.abs() * w).T @ vd.abs()
        x = min(abs(g[h].item()) * S, 104)
        tol = state_tolerance(S, D, H, dtype, x) * mag + 1e-37
        assert ((s[0, h].double() - want).abs() <= tol).all()


def test_a_compiled_training_step_of_the_layer(device):
    """Forward and gradients through the training compiler: the same ops in the same order, so the values are equal."""
    from xpu_graph_amd import mi355x_compiler

    _xops().enable_autograd()
    B, S, H, D = 2, 100, 2, 64
    bf = torch.bfloat16
    ang = torch.rand(S, D // 2, generator=torch.Generator().manual_seed(0)) * 6
    cos, sin, g = ang.cos().to(device), ang.sin().to(device), decays(H, device, "model")
    pos = torch.arange(S, device=device)
    n = torch.tensor([S, 61], device=device)

    def attend(q, k, v, wq, wk, state):
        q, k = torch.ops.xpu_ops.qk_norm_rope(q, k, wq, wk, cos, sin, pos, [], False, 1e-6)
        q = torch.ops.xpu_ops.rope_axes(q, cos, sin, pos, [])
        return torch.ops.xpu_ops.linear_attn(q, k, v, g, state, n, D**-0.5)

    def inputs(seed):
        x = [make((B, H, S, D), bf, device, seed + i) for i in range(3)]
        x += [(1 + 0.1 * torch.randn(D, device=device)).to(bf) for _ in range(2)] + [torch.randn(B, H, D, D, device=device)]
        return [t.requires_grad_() for t in x]

    step = torch.compile(attend, backend=mi355x_compiler(is_training=True), dynamic=False)
    for seed in (0, 10):
        leaves = inputs(seed)
        up = make((B, H, S, D), bf, device, seed + 7), torch.randn(B, H, D, D, device=device)
        want, got = attend(*leaves), step(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        want, got = (torch.autograd.grad(y, leaves, up) for y in (want, got))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
