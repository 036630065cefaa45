"""Cases and plain forms of the operators that prepare queries and keys (rotary positions with several axes, per-head
norm with rotation) and of linear attention with a decay for each head (prompt, training, single token).

`run` computes each operator from elementary torch operations in 32 bits, or, where `own` is set, through
`torch.ops.xpu_ops`; `exact` evaluates the definitions token by token in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_CHUNK = 64


def listed():
    return [
        # a short sequence with text and one small image, fine-tuned: latency of a call and of its backward, part of the head rotated
        {"name": "axes_few", "op": "rope_axes", "B": 1, "S": 67, "H": 4, "D": 64, "R": 32, "axes": 3, "woven": False, "dtype": "f16", "train": True},
        # a batch of two requests with images of several thousand patches each
        {"name": "axes_image", "op": "rope_axes", "B": 2, "S": 6144, "H": 32, "D": 128, "R": 128, "axes": 3, "woven": True, "dtype": "bf16", "train": False},
        # a decode step: one new token of eight sequences, shared key heads
        {"name": "prep_token", "op": "qk_norm_rope", "B": 8, "S": 1, "H": 32, "Hkv": 8, "D": 128, "R": 128, "axes": 1, "woven": False, "dtype": "bf16", "train": False},
        # a prompt batch of the benchmark's decoder block, read out of the packed projection
        {"name": "prep_prompt", "op": "qk_norm_rope", "B": 4, "S": 2048, "H": 32, "Hkv": 8, "D": 128, "R": 128, "axes": 1, "woven": False, "dtype": "bf16", "train": False},
        # the same block in training: forward and the gradients of q, k and both weights
        {"name": "prep_train", "op": "qk_norm_rope", "B": 4, "S": 2048, "H": 32, "Hkv": 32, "D": 128, "R": 128, "axes": 1, "woven": False, "dtype": "bf16", "train": True},
        # training on images with an odd length, a head size that is no power of two and three positions a token
        {"name": "prep_odd", "op": "qk_norm_rope", "B": 3, "S": 1371, "H": 10, "Hkv": 5, "D": 96, "R": 96, "axes": 3, "woven": False, "dtype": "f16", "train": True},
        # a small ragged prompt batch that continues from cached states
        {"name": "lin_short", "op": "linear_attn", "B": 3, "S": 97, "H": 8, "Hkv": 8, "D": 64, "ragged": True, "state": True, "dtype": "f16", "train": False},
        # one long document
        {"name": "lin_long", "op": "linear_attn", "B": 1, "S": 32768, "H": 32, "Hkv": 32, "D": 128, "ragged": False, "state": False, "dtype": "bf16", "train": False},
        # training of the benchmark's block size
        {"name": "lin_train", "op": "linear_attn", "B": 4, "S": 2048, "H": 32, "Hkv": 32, "D": 128, "ragged": False, "state": False, "dtype": "bf16", "train": True},
        # training on padded sequences with shared key heads and a learned initial state
        {"name": "lin_train_odd", "op": "linear_attn", "B": 2, "S": 1023, "H": 12, "Hkv": 4, "D": 64, "ragged": True, "state": True, "dtype": "f16", "train": True},
        # decoding a single sequence
        {"name": "step_one", "op": "linear_attn_step", "B": 1, "H": 32, "Hkv": 32, "D": 128, "dtype": "bf16"},
        # decoding a full serving batch, shared key heads
        {"name": "step_batch", "op": "linear_attn_step", "B": 64, "H": 32, "Hkv": 8, "D": 128, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One case of the ranges above; sizes by their logarithm, under the cost of the largest listed case of its kind."""
    op = rng.choice(["rope_axes", "qk_norm_rope", "linear_attn", "linear_attn_step"])
    dtype = rng.choice(["bf16", "f16"])
    if op in ("rope_axes", "qk_norm_rope"):
        D = rng.choice([64, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, 16 * rng.randint(1, D // 16)])
        axes = rng.choice([1, 3]) if op == "qk_norm_rope" else rng.choice([2, 3])
        Hkv = rng.randint(1, 8)
        H = Hkv * rng.randint(1, 4)
        B, train = rng.randint(1, 8), rng.random() < 0.5
        most = (25_000_000 if train else 40_000_000) // (B * (H + Hkv) * D)
        S = min(_between(rng, 1, 8192), max(1, most))
        case = {"op": op, "B": B, "S": S, "H": H, "D": D, "R": R, "axes": axes, "woven": axes > 1 and rng.random() < 0.5, "dtype": dtype, "train": train}
        return {**case, "Hkv": Hkv} if op == "qk_norm_rope" else case
    D = rng.choice([64, 128])
    Hkv = rng.randint(1, 16)
    H = Hkv * rng.choice([1, 1, 2, 4])
    if op == "linear_attn_step":
        return {"op": op, "B": min(_between(rng, 1, 128), 2048 * 64 // (H * D) or 1), "H": H, "Hkv": Hkv, "D": D, "dtype": dtype}
    B, train = rng.randint(1, 6), rng.random() < 0.5
    most = (30_000_000 if train else 100_000_000) // (B * H * D)
    S = max(1, min(_between(rng, 1, 16384), most))
    return {"op": op, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D, "ragged": rng.random() < 0.5, "state": rng.random() < 0.5, "dtype": dtype, "train": train}


# ------------------------------------------------------------------ inputs
def _sections(case):
    """Pairs per axis: the first axis takes a little less than its share, as time does beside height and width."""
    half, axes = case["R"] // 2, case["axes"]
    if axes == 1:
        return [half]
    first = half - (axes - 1) * ((half + 1) // axes)
    if first < 0:
        first = half % axes
    rest = half - first
    return [first] + [rest // (axes - 1) + (1 if i < rest % (axes - 1) else 0) for i in range(axes - 1)]


def _positions(case, dev, gen):
    """[axes, B, S]: a text prefix that counts alike on every axis, then a grid of patches; a decode step stands anywhere."""
    B, S, axes = case["B"], case["S"], case["axes"]
    first = torch.randint(0, 4096, (B, 1), device=dev, generator=gen)
    t = torch.arange(S, device=dev).expand(B, S)
    if axes == 1:
        return (first + t)[None].contiguous()
    text, wide = S // 4, max(1, int(math.sqrt(S)))
    high = max(1, wide // 2)
    idx = (t - text).clamp_min(0)
    grid = [idx // (high * wide), (idx // wide) % high, idx % wide][-axes:]
    return torch.stack([first + torch.where(t < text, t, text + g) for g in grid])


def _tables(case, count, dev):
    half = case["R"] // 2
    inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    angle = torch.arange(count, device=dev, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _log_decay(H, dev):
    """From a memory of two tokens to one of a thousand, over the heads."""
    return -torch.exp2(-1.0 - 9.0 * torch.arange(H, device=dev, dtype=torch.float32) / max(H - 1, 1))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt, op, B, H, D = _DTYPES[case["dtype"]], case["op"], case["B"], case["H"], case["D"]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, device=dev, generator=gen, dtype=torch.float32).to(dtype)

    s = {"case": case}
    if op in ("rope_axes", "qk_norm_rope"):
        S, Hkv = case["S"], case.get("Hkv", 0)
        packed = randn(B, S, (H + 2 * Hkv) * D)  # what the projection leaves: queries, keys, values side by side
        heads = packed.view(B, S, H + 2 * Hkv, D).transpose(1, 2)
        s["q"], s["positions"] = heads[:, :H], _positions(case, dev, gen)
        s["cos"], s["sin"] = _tables(case, 4096 + S, dev)
        s["sections"], s["eps"] = _sections(case), 1e-6
        if case["train"]:
            s["gq"] = randn(B, S, H, D).transpose(1, 2)
        if Hkv:
            s["k"] = heads[:, H : H + Hkv]
            s["wq"], s["wk"] = (1 + 0.1 * randn(D).float()).to(dt), (1 + 0.1 * randn(D).float()).to(dt)
            if case["train"]:
                s["gk"] = randn(B, S, Hkv, D).transpose(1, 2)
        if case["train"]:
            for name in ("q", "k", "wq", "wk"):
                if name in s:
                    s[name] = s[name].detach().requires_grad_()
        return s
    Hkv = case["Hkv"]
    S = case.get("S", 1)
    q, k, v = randn(B, S, H, D), randn(B, S, Hkv, D), randn(B, S, Hkv, D)
    s["q"], s["k"], s["v"] = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    s["log_decay"], s["scale"] = _log_decay(H, dev), D**-0.5
    s["state"] = s["lengths"] = None
    if op == "linear_attn_step" or case["state"]:
        s["state"] = randn(B, H, D, D, dtype=torch.float32)
    if op == "linear_attn" and case["ragged"]:
        s["lengths"] = torch.randint((S + 1) // 2, S + 1, (B,), device=dev, generator=gen)
    if case.get("train"):
        s["d_out"], s["d_state"] = randn(B, S, H, D).transpose(1, 2), 0.1 * randn(B, H, D, D, dtype=torch.float32)
        for name in ("q", "k", "v", "state"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# -------------------------------------------------- the rotations, in 32 bits
def _pair_axes(sections, woven):
    """The axis that turns each pair: runs of pairs, or the axes in turn as long as each has pairs left."""
    if not woven:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    A = len(sections)
    return [i % A if i < A * sections[i % A] else 0 for i in range(sum(sections))]


def _angles(s):
    """cos and sin of every pair of every token, [B, 1, S, R/2]."""
    axis = torch.tensor(_pair_axes(s["sections"], s["case"]["woven"]), device=s["positions"].device)
    at = s["positions"][axis].permute(1, 2, 0)
    pair = torch.arange(len(axis), device=at.device)
    return s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]


def _turn(x, cos, sin, R):
    a, b = x[..., : R // 2], x[..., R // 2 : R]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], -1)


def _norm(x, eps):
    xf = x.float()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
    return xf * r, r


def _norm_turn_back(gy, x, w, cos, sin, R, eps):
    xhat, r = _norm(x, eps)
    gn = _turn(gy.float(), cos, -sin, R)
    gw = (gn * xhat).sum((0, 1, 2))
    gx = gn * w.float()
    return (r * (gx - xhat * (gx * xhat).mean(-1, keepdim=True))).to(x.dtype), gw.to(w.dtype)


def _plain_prepare(s):
    case, R, eps = s["case"], s["case"]["R"], s["eps"]
    with torch.no_grad():
        cos, sin = _angles(s)
        if case["op"] == "rope_axes":
            out = {"y": _turn(s["q"].float(), cos, sin, R).to(s["q"].dtype)}
            if case["train"]:
                out["gx"] = _turn(s["gq"].float(), cos, -sin, R).to(s["q"].dtype)
            return out
        out = {"q": _turn(_norm(s["q"], eps)[0] * s["wq"].float(), cos, sin, R).to(s["q"].dtype)}
        out["k"] = _turn(_norm(s["k"], eps)[0] * s["wk"].float(), cos, sin, R).to(s["k"].dtype)
        if case["train"]:
            out["gq"], out["gwq"] = _norm_turn_back(s["gq"], s["q"], s["wq"], cos, sin, R, eps)
            out["gk"], out["gwk"] = _norm_turn_back(s["gk"], s["k"], s["wk"], cos, sin, R, eps)
        return out


# -------------------------------------------- linear attention, in 32 bits
def _decayed(g, n):
    """exp(g * n) for the heads' log decays g [H] and whole numbers n, [H, *n.shape]; 0 where n < 0."""
    e = g.view(-1, *([1] * n.dim())) * n.float()
    return torch.where(n >= 0, torch.exp(torch.where(n >= 0, e, 0.0)), 0.0)


def _chunks(t):
    B, H, S, D = t.shape
    n = -(-S // _CHUNK)
    return torch.nn.functional.pad(t, (0, 0, 0, n * _CHUNK - S)).view(B, H, n, _CHUNK, D)


def _scan(q, k, v, g, state):
    """sum over s <= t of decay^(t - s) (q_t . k_s) v_s + decay^(t + 1) q_t state, by chunks."""
    B, H, S, D = q.shape
    qc, kc, vc = _chunks(q), _chunks(k), _chunks(v)
    n = qc.shape[2]
    i = torch.arange(_CHUNK, device=q.device)
    inside = (qc @ kc.transpose(-1, -2)) * _decayed(g, i[:, None] - i)[:, None]
    out = inside @ vc
    own_states = ((kc * _decayed(g, _CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2) @ vc).view(B, H, n, D * D)
    c = torch.arange(n, device=q.device)
    before = _decayed(g * _CHUNK, c[:, None] - 1 - c) @ own_states
    if state is not None:
        before = before + _decayed(g * _CHUNK, c)[..., None] * state.view(B, H, 1, D * D)
    out = out + _decayed(g, i + 1)[:, None, :, None] * (qc @ before.view(B, H, n, D, D))
    return out.view(B, H, n * _CHUNK, D)[:, :, :S]


def _plain_linear(s):
    case, g, scale = s["case"], s["log_decay"], s["scale"]
    with torch.no_grad():
        dt, group = s["q"].dtype, case["H"] // case["Hkv"]
        B, H, S, D = s["q"].shape
        length = s["lengths"] if s["lengths"] is not None else torch.full((B,), S, device=g.device)
        t = torch.arange(S, device=g.device)
        alive = (t < length[:, None])[:, None, :, None]
        wide = lambda x: x.float().repeat_interleave(group, 1)  # noqa: E731
        clean = lambda x: torch.where(alive, x, 0.0)  # noqa: E731
        q, k, v = clean(s["q"].float()), clean(wide(s["k"])), clean(wide(s["v"]))
        state = s["state"]
        out = {"o": (scale * _scan(q, k, v, g, state)).to(dt)}
        out["o"] = torch.where(alive, out["o"], torch.zeros((), dtype=dt, device=g.device))
        left = _decayed(g, length[:, None] - 1 - t).transpose(0, 1)[..., None]  # [B, H, S, 1]
        whole = _decayed(g, length).transpose(0, 1)[..., None, None]
        out["state"] = (k * left).transpose(-1, -2) @ v
        if state is not None:
            out["state"] = out["state"] + whole * state
        if case["train"]:
            go, ds = clean(s["d_out"].float()), s["d_state"]
            back = lambda x: x.flip(2)  # noqa: E731
            gq = scale * _scan(go, v, k, g, state.transpose(-1, -2).contiguous() if state is not None else None)
            gk = scale * back(_scan(back(v), back(go), back(q), g, None)) + left * (v @ ds.transpose(-1, -2))
            gv = scale * back(_scan(back(k), back(q), back(go), g, None)) + left * (k @ ds)
            narrow = lambda x: clean(x).view(B, H // group, group, S, D).sum(2)  # noqa: E731
            out["gq"], out["gk"], out["gv"] = clean(gq).to(dt), narrow(gk).to(dt), narrow(gv).to(dt)
            if state is not None:
                reached = _decayed(g, t + 1)[:, :, None]
                out["gs"] = scale * ((q * reached).transpose(-1, -2) @ go) + whole * ds
        return out


def _plain_step(s):
    group = s["case"]["H"] // s["case"]["Hkv"]
    wide = lambda x: x.float().repeat_interleave(group, 1)  # noqa: E731
    k, v = wide(s["k"]), wide(s["v"])
    state = s["state"].mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k.transpose(-1, -2) * v)
    return {"o": (s["scale"] * (s["q"].float() @ state)).to(s["q"].dtype), "state": state}


# ----------------------------------------------------------------- one pass
def _own_prepare(s):
    import xpu_graph_amd.ops as xops

    case, ops = s["case"], torch.ops.xpu_ops
    turn = (s["cos"], s["sin"], s["positions"], s["sections"], case["woven"])
    if case["train"]:
        xops.enable_autograd()
    if case["op"] == "rope_axes":
        y = ops.rope_axes(s["q"], *turn)
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "gx": torch.autograd.grad(y, s["q"], s["gq"])[0]}
    q, k = ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], *turn, s["eps"])
    if not case["train"]:
        return {"q": q, "k": k}
    gq, gk, gwq, gwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return {"q": q.detach(), "k": k.detach(), "gq": gq, "gk": gk, "gwq": gwq, "gwk": gwk}


def _own_linear(s):
    import xpu_graph_amd.ops as xops

    case, ops = s["case"], torch.ops.xpu_ops
    if case["op"] == "linear_attn_step":
        return {"o": ops.linear_attn_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["scale"]), "state": s["state"]}
    if case["train"]:
        xops.enable_autograd()
    o, state = ops.linear_attn(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["lengths"], s["scale"])
    if not case["train"]:
        return {"o": o, "state": state}
    leaves = [s[n] for n in ("q", "k", "v", "state") if s[n] is not None]
    grads = torch.autograd.grad((o, state), leaves, (s["d_out"], s["d_state"]))
    return {"o": o.detach(), "state": state.detach(), **dict(zip(("gq", "gk", "gv", "gs"), grads))}


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_prepare(state) if op in ("rope_axes", "qk_norm_rope") else _own_linear(state)
    if op in ("rope_axes", "qk_norm_rope"):
        return _plain_prepare(state)
    return _plain_step(state) if op == "linear_attn_step" else _plain_linear(state)


def work(case):
    op, B, H, D = case["op"], case["B"], case["H"], case["D"]
    if op in ("rope_axes", "qk_norm_rope"):
        n, norm = B * case["S"] * (H + case.get("Hkv", 0)) * D, 4 if op == "qk_norm_rope" else 0
        tables = 8 * case["axes"] * B * case["S"] + 4 * B * case["S"] * case["R"]
        passes = 2 + ((3 if norm else 2) if case["train"] else 0)
        return {"bytes": 2 * n * passes + tables, "flops": n * (3 + norm) * (3 if case["train"] else 1)}
    Hkv, state = case["Hkv"], 4 * B * H * D * D
    if op == "linear_attn_step":
        return {"bytes": 2 * state + 2 * B * D * (2 * H + 2 * Hkv), "flops": 5 * B * H * D * D}
    token = 2 * B * case["S"] * D
    states = state * (2 if case["state"] else 1)
    if not case["train"]:
        return {"bytes": token * (2 * H + 2 * Hkv) + states, "flops": 4 * B * case["S"] * H * D * D}
    bytes_ = token * (2 * H + 2 * Hkv) + token * (3 * H + 4 * Hkv) + states + state * (2 if case["state"] else 1)
    return {"bytes": bytes_, "flops": 14 * B * case["S"] * H * D * D}


# ------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = {n: x.detach() if isinstance(x, torch.Tensor) else x for n, x in prepare(case, seed).items()}

    def prepared():
        R, half = case["R"], case["R"] // 2
        rows = s["positions"].double()
        y = {}

        def rotated(x, back):
            out = x.clone()
            for i, a in enumerate(_pair_axes(s["sections"], case["woven"])):
                at = rows[a].long()
                c, n = s["cos"][at, i].double()[:, None], s["sin"][at, i].double()[:, None]
                n = -n if back else n
                out[..., i] = x[..., i] * c - x[..., i + half] * n
                out[..., i + half] = x[..., i] * n + x[..., i + half] * c
            return out

        if case["op"] == "rope_axes":
            y["y"] = rotated(s["q"].double(), False)
            if case["train"]:
                y["gx"] = rotated(s["gq"].double(), True)
            return y
        for name in ("q", "k"):
            x, w = s[name].double(), s["w" + name].double()
            size = (x.pow(2).sum(-1, keepdim=True) / case["D"] + s["eps"]).sqrt()
            y[name] = rotated(x / size * w, False)
            if case["train"]:
                gn = rotated(s["g" + name].double(), True)
                y["gw" + name] = torch.einsum("bhsd,bhsd->d", gn, x / size)
                gw = gn * w
                y["g" + name] = gw / size - x * (gw * x).sum(-1, keepdim=True) / (case["D"] * size.pow(3))
        return y

    def recurrence():
        group, scale = case["H"] // case["Hkv"], s["scale"]
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        B, H, S, D = q.shape
        lam = s["log_decay"].double().exp()[:, None, None]
        state = s["state"].double().clone() if s["state"] is not None else q.new_zeros(B, H, D, D)
        length = s["lengths"] if s["lengths"] is not None else torch.full((B,), S, device=q.device)
        alive = torch.arange(S, device=q.device) < length[:, None]
        o = torch.zeros_like(q)
        train = bool(case.get("train"))
        gq = torch.zeros_like(q)
        for t in range(S):
            live = alive[:, t].view(B, 1, 1, 1)
            new = state * lam + k[:, :, t, :, None] * v[:, :, t, None, :]
            state = torch.where(live, new, state) if s["lengths"] is not None else new
            o[:, :, t] = torch.where(live[..., 0], scale * (q[:, :, t, None] @ state)[:, :, 0], 0.0)
            if train:
                go = s["d_out"][:, :, t].double()
                gq[:, :, t] = torch.where(live[..., 0], scale * (state @ go[..., None])[..., 0], 0.0)
        y = {"o": o, "state": state}
        if train:
            gk, gv, big = torch.zeros_like(q), torch.zeros_like(q), s["d_state"].double()
            for t in range(S - 1, -1, -1):
                live = alive[:, t].view(B, 1, 1, 1)
                here = big + scale * q[:, :, t, :, None] * s["d_out"][:, :, t, None, :].double()
                gk[:, :, t] = torch.where(live[..., 0], (here @ v[:, :, t, :, None])[..., 0], 0.0)
                gv[:, :, t] = torch.where(live[..., 0], (k[:, :, t, None] @ here)[:, :, 0], 0.0)
                big = torch.where(live, lam * here, big)
            narrow = lambda x: x.view(B, H // group, group, S, D).sum(2)  # noqa: E731
            y.update(gq=gq, gk=narrow(gk), gv=narrow(gv))
            if s["state"] is not None:
                y["gs"] = big
        return y

    with torch.no_grad():
        return prepared() if case["op"] in ("rope_axes", "qk_norm_rope") else recurrence()
