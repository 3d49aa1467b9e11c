"""The operators of a differential-attention layer stack: rotary positions, differential attention, and the norms before and after a
block with its gate and residual scale.

Every case is a pass through one operator: `run` computes it from elementary torch operations, or, where `own` is true, through
`rectools_amd.ops`.  Rows are the framework's: float32, `[rows, heads * columns]`, sessions packed behind each other (`cu`) or padded to a
window, item id 0 = padding.
"""
from __future__ import annotations

import math
import random
import typing as tp

import torch

own = False

DEV = "cuda"


# ---- the cases ------------------------------------------------------------------------------------------------------------------------
def listed() -> tp.List[dict]:
    return [
        # the newest item of 64 sessions: queries and keys of one row each, before they meet the stored keys
        dict(name="rotary, newest rows", op="rotary", rows=64, heads=8, kv_heads=8, hd=32, rot=32, interleaved=False, far=False,
             scaling="none", train=False),
        # the rows of a training batch (128 sessions of a 200 window, d = 256): queries and keys, forward and backward
        dict(name="rotary, session batch", op="rotary", rows=17_920, heads=8, kv_heads=8, hd=32, rot=32, interleaved=False, far=False,
             scaling="none", train=True),
        # long histories behind position 900,000, half of each head rotated, frequencies scaled by parts, shared key heads
        dict(name="rotary, far positions", op="rotary", rows=65_536, heads=16, kv_heads=4, hd=64, rot=32, interleaved=True, far=True,
             scaling="parts", train=False),
        # one row per session in recommend(): the final block's residual
        dict(name="norms, newest rows", op="norms", rows=256, d=256, kind="rms", gate=True, scale=True, post=True, pre=True, alpha=1.0,
             train=False),
        # the rows of a padded training batch (128 x 200, d = 256), LayerNorm with biases
        dict(name="norms, session batch", op="norms", rows=25_600, d=256, kind="layer", gate=True, scale=True, post=True, pre=True,
             alpha=1.0, train=True),
        # n_factors = 50: rows that no vector load divides
        dict(name="norms, 50 factors", op="norms", rows=40_001, d=50, kind="rms", gate=True, scale=True, post=True, pre=True, alpha=1.0,
             train=True),
        # a wide residual stream
        dict(name="norms, wide rows", op="norms", rows=16_384, d=2_048, kind="rms", gate=True, scale=True, post=True, pre=True, alpha=1.5,
             train=True),
        # recommend(): the last query of every session against its own rows
        dict(name="attention, last queries", op="attention", B=1_024, L=200, lens=1, q_rows=1, heads=4, kv_heads=4, hd=32, causal=True,
             padded=False, train=False),
        # a few very long sessions, one query each, shared key heads
        dict(name="attention, long keys", op="attention", B=8, L=65_536, lens=2, q_rows=1, heads=8, kv_heads=2, hd=64, causal=True,
             padded=False, train=False),
        # the training step's packed sessions (d = 256, 4 heads)
        dict(name="attention, session batch", op="attention", B=128, L=200, lens=3, q_rows=0, heads=4, kv_heads=4, hd=32, causal=True,
             padded=False, train=True),
        # n_factors = 50 with one head: 25 query columns, padded windows of 100 with masked keys, both directions visible
        dict(name="attention, 50 factors", op="attention", B=128, L=100, lens=4, q_rows=0, heads=1, kv_heads=1, hd=25, causal=False,
             padded=True, train=True),
        # two long sessions at d = 512
        dict(name="attention, long sessions", op="attention", B=2, L=4_096, lens=0, q_rows=0, heads=4, kv_heads=4, hd=64, causal=True,
             padded=False, train=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["rotary", "norms", "attention", "attention"])
    if op == "rotary":
        hd = rng.randint(4, 128)
        rot = 2 * rng.randint(1, hd // 2)
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2, 4])
        rows = _log(rng, 1, min(131_072, 65_536 * 20 * 64 // ((heads + kv) * hd)))
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv, hd=hd, rot=rot, interleaved=rng.random() < 0.5, far=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "base", "parts"]), train=rng.random() < 0.5)
    if op == "norms":
        d = _log(rng, 16, 4_096)
        return dict(op=op, rows=_log(rng, 1, min(200_000, 16_384 * 2_048 // d)), d=d, kind=rng.choice(["rms", "layer"]),
                    gate=rng.random() < 0.7, scale=rng.random() < 0.7, post=rng.random() < 0.8, pre=rng.random() < 0.8,
                    alpha=rng.choice([1.0, 1.25]), train=rng.random() < 0.6)
    hd = rng.randint(4, 64)
    kv = rng.choice([1, 2, 4])
    heads = kv * rng.choice([1, 1, 2])
    if rng.random() < 0.4:      # the newest rows of stored sessions
        q_rows = rng.choice([1, 1, 1, 5])
        L = _log(rng, max(2, q_rows), 65_536)
        B = _log(rng, 1, max(1, min(2_048, 400_000 // L)))
        return dict(op=op, B=B, L=L, lens=rng.randint(1, 999), q_rows=q_rows, heads=heads, kv_heads=kv, hd=hd, causal=True, padded=False,
                    train=False)
    L = _log(rng, 1, 4_096)
    B = _log(rng, 1, max(1, min(256, 2 * 4_096 * 4_096 * 4 // (L * L * heads), 40_000 // L)))
    return dict(op=op, B=B, L=L, lens=rng.randint(1, 999), q_rows=0, heads=heads, kv_heads=kv, hd=hd, causal=rng.random() < 0.7,
                padded=rng.random() < 0.4, train=rng.random() < 0.7)


def _lengths(case: dict) -> tp.List[int]:
    """Session lengths: all equal to the window (lens = 0), or long-tailed and cut at it, as interaction histories are."""
    B, L = case["B"], case["L"]
    if case["lens"] == 0:
        return [L] * B
    rng = random.Random(case["lens"])
    low = max(1, case["q_rows"])
    return [max(low, min(L, int(L * 0.6 * math.exp(rng.gauss(0.0, 0.8))))) for _ in range(B)]


def _pairs(case: dict) -> int:
    """(query, visible key) pairs of one head."""
    n = 0
    for m in _lengths(case):
        if case["q_rows"]:
            q = case["q_rows"]
            n += q * (m - q) + q * (q + 1) // 2
        elif case["padded"]:      # every row of the window asks; the m real keys (the window's last ones) can be seen
            n += m * (m + 1) // 2 if case["causal"] else case["L"] * m
        else:
            n += m * (m + 1) // 2 if case["causal"] else m * m
    return n


def work(case: dict) -> tp.Dict[str, float]:
    if case["op"] == "rotary":
        cols = (case["heads"] + case["kv_heads"]) * case["hd"]
        turned = (case["heads"] + case["kv_heads"]) * case["rot"]
        passes = 2 if case["train"] else 1
        return {"bytes": case["rows"] * (passes * 2 * cols * 4 + 8), "flops": passes * case["rows"] * turned * 3}
    if case["op"] == "norms":
        n = case["rows"] * case["d"]
        ins, outs = 2 + case["gate"], 1 + case["pre"]
        fwd = (ins + outs) * 4 * n
        if not case["train"]:
            return {"bytes": fwd, "flops": 14 * n}
        return {"bytes": fwd + (outs + ins) * 4 * n, "flops": 44 * n}      # the outputs' gradients read, the inputs' written
    lens, hd, H, Hk = _lengths(case), case["hd"], case["heads"], case["kv_heads"]
    keys = case["B"] * case["L"] if case["padded"] else sum(lens)
    rows = case["B"] * case["q_rows"] if case["q_rows"] else keys
    q, kv = rows * H * 2 * hd, keys * Hk * 4 * hd
    moved = 4 * (2 * q + kv)
    flops = _pairs(case) * H * 8 * hd      # two maps of hd columns, one product of their difference with 2 hd columns
    if case["train"]:
        moved += 4 * (2 * q + kv)
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _frequencies(rot: int, scaling: str) -> torch.Tensor:
    """Radians per position of every pair, float64 (base 10,000; windows four times the trained 4,096 positions)."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base, factor, trained = 10_000.0, 4.0, 4_096.0
    if scaling == "base" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":      # pairs that turn often keep their frequency, slow ones are stretched, a ramp between
        turns = trained * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed * 1_000_003 + 17)
    rnd = lambda *shape, s=1.0: torch.randn(shape, generator=g, device=DEV) * s      # noqa: E731
    train = case["train"]
    leaf = lambda t: t.requires_grad_(train)      # noqa: E731
    st: tp.Dict[str, tp.Any] = {"case": case}
    if case["op"] == "rotary":
        M, hd = case["rows"], case["hd"]
        st["q"], st["k"] = leaf(rnd(M, case["heads"] * hd)), leaf(rnd(M, case["kv_heads"] * hd))
        if case["far"]:
            st["pos"] = torch.arange(M, device=DEV) + 900_000
        else:
            st["pos"] = torch.randint(0, 200, (M,), generator=g, device=DEV)
        st["freq"] = _frequencies(case["rot"], case["scaling"]).to(DEV)
        st["gain"] = 0.1 * math.log(4.0) + 1.0 if case["scaling"] == "parts" else 1.0
        if train:
            st["gq"], st["gk"] = rnd(M, case["heads"] * hd, s=0.01), rnd(M, case["kv_heads"] * hd, s=0.01)
        return st
    if case["op"] == "norms":
        M, d = case["rows"], case["d"]
        st["x"], st["f"] = leaf(rnd(M, d, s=2.0)), leaf(rnd(M, d, s=0.5) + 0.1)
        layer = case["kind"] == "layer"
        st["z"] = leaf(rnd(M, d)) if case["gate"] else None
        st["s"] = leaf(0.5 + rnd(d, s=0.2)) if case["scale"] else None
        st["pw"] = leaf(1.0 + rnd(d, s=0.1)) if case["post"] else None
        st["pb"] = leaf(rnd(d, s=0.1)) if case["post"] and layer else None
        st["nw"] = leaf(1.0 + rnd(d, s=0.1)) if case["pre"] else None
        st["nb"] = leaf(rnd(d, s=0.1)) if case["pre"] and layer else None
        if train:
            st["gx"], st["gh"] = rnd(M, d, s=0.01), rnd(M, d, s=0.01) if case["pre"] else None
        return st
    hd, H, Hk, B, L = case["hd"], case["heads"], case["kv_heads"], case["B"], case["L"]
    lens = torch.tensor(_lengths(case))
    if case["padded"]:
        rows = keys = B * L
        ids = torch.randint(1, 1_000, (B, L), generator=g, device=DEV)
        ids[torch.arange(L, device=DEV)[None] < (L - lens.to(DEV))[:, None]] = 0
        st["ids"], st["cu_q"], st["cu_k"] = ids.reshape(-1), None, None
        st["Lq"] = L
    else:
        cu = torch.zeros(B + 1, dtype=torch.int64)
        cu[1:] = lens.cumsum(0)
        keys = int(cu[-1])
        st["ids"], st["cu_k"] = None, cu.to(DEV)
        st["Lq"] = case["q_rows"] or L
        rows = B * case["q_rows"] if case["q_rows"] else keys
        st["cu_q"] = None if case["q_rows"] else st["cu_k"]
    st["q"], st["k"] = leaf(rnd(rows, H * 2 * hd, s=1.2)), leaf(rnd(keys, Hk * 2 * hd))
    st["v"] = leaf(rnd(keys, Hk * 2 * hd))
    st["lq1"], st["lk1"], st["lq2"], st["lk2"] = (leaf(rnd(H, hd, s=0.1)) for _ in range(4))
    st["w"] = leaf(1.0 + rnd(2 * hd, s=0.1))
    st["init"] = 0.8 - 0.6 * math.exp(-0.3)
    if train:
        st["gy"] = rnd(rows, H * 2 * hd, s=0.01)
    return st


# ---- plain forms ----------------------------------------------------------------------------------------------------------------------
def _turn(x: torch.Tensor, st: dict, heads: int) -> torch.Tensor:
    case = st["case"]
    rot, M = case["rot"], x.shape[0]
    angle = st["pos"].double()[:, None] * st["freq"][None]
    cos, sin = ((angle.cos() * st["gain"]).float()[:, None], (angle.sin() * st["gain"]).float()[:, None])
    x = x.view(M, heads, case["hd"])
    part, rest = x[..., :rot], x[..., rot:]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        out = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(M, heads, rot)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        out = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((out, rest), -1).reshape(M, -1)


def _norm(x: torch.Tensor, w: torch.Tensor, b: tp.Optional[torch.Tensor], kind: str) -> torch.Tensor:
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    return x * w if b is None else x * w + b


def _plain_norms(st: dict) -> tp.Tuple[torch.Tensor, tp.Optional[torch.Tensor]]:
    case = st["case"]
    n = _norm(st["f"], st["pw"], st["pb"], case["kind"]) if case["post"] else st["f"]
    if case["gate"]:
        n = n / (1.0 + torch.exp(-st["z"]))
    if case["scale"]:
        n = n * st["s"]
    y = case["alpha"] * st["x"] + n
    return y, _norm(y, st["nw"], st["nb"], case["kind"]) if case["pre"] else None


def _windows(st: dict, x: torch.Tensor, cu: tp.Optional[torch.Tensor], n: int, parts: int, cols: int) -> torch.Tensor:
    """[B, parts, n, cols]: the rows of every session, the last one at the window's end; places without a row read the session's first."""
    B = st["case"]["B"]
    if cu is None:
        return x.view(B, n, parts, cols).transpose(1, 2)
    at = cu[1:, None] - n + torch.arange(n, device=x.device)[None]
    return x.index_select(0, torch.maximum(at, cu[:-1, None]).reshape(-1)).view(B, n, parts, cols).transpose(1, 2)


def _plain_attention(st: dict) -> torch.Tensor:
    case = st["case"]
    B, L, H, Hk, hd, n = case["B"], case["L"], case["heads"], case["kv_heads"], case["hd"], st["Lq"]
    share = torch.arange(H, device=DEV) // (H // Hk)
    q = _windows(st, st["q"], st["cu_q"], n, 2 * H, hd).reshape(B, H, 2, n, hd)
    k = _windows(st, st["k"], st["cu_k"], L, 2 * Hk, hd).reshape(B, Hk, 2, L, hd)[:, share]
    v = _windows(st, st["v"], st["cu_k"], L, Hk, 2 * hd)[:, share]
    at_k = torch.arange(L, device=DEV)[None, None]
    if case["padded"]:
        seen = (st["ids"].view(B, 1, L) != 0).expand(B, n, L)
    else:
        seen = (at_k >= L - (st["cu_k"][1:] - st["cu_k"][:-1])[:, None, None]).expand(B, n, L)
    if case["causal"]:
        seen = seen & (at_k <= torch.arange(n, device=DEV)[None, :, None] + (L - n))
    seen = seen[:, None, None]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True).detach()
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    a = e / torch.where(total > 0, total, 1.0)
    lam = torch.exp((st["lq1"] * st["lk1"]).sum(-1)) - torch.exp((st["lq2"] * st["lk2"]).sum(-1)) + st["init"]
    o = torch.matmul(a[:, :, 0] - lam[:, None, None] * a[:, :, 1], v)
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + 1e-5) * st["w"] * (1.0 - st["init"])
    o = o.transpose(1, 2)      # [B, n, H, 2 hd], the sessions' rows at the windows' ends
    if st["cu_q"] is None:
        return o.reshape(B * n, -1)
    at_q = torch.arange(n, device=DEV)[None]
    return o[at_q >= n - (st["cu_q"][1:] - st["cu_q"][:-1])[:, None]].reshape(st["q"].shape[0], -1)


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def _forward(st: dict) -> tp.Dict[str, torch.Tensor]:
    case = st["case"]
    if own:
        from rectools_amd import ops
    if case["op"] == "rotary":
        if own:
            q, k = ops.rotary_qk(st["q"], st["k"], st["pos"], st["freq"], case["heads"], case["kv_heads"], case["interleaved"], st["gain"])
        else:
            q, k = _turn(st["q"], st, case["heads"]), _turn(st["k"], st, case["kv_heads"])
        return {"q": q, "k": k}
    if case["op"] == "norms":
        if own:
            y, h = ops.norm_gate_residual(st["x"], st["f"], gate=st["z"], post=(st["pw"], st["pb"]) if case["post"] else None, scale=st["s"],
                                          pre=(st["nw"], st["nb"]) if case["pre"] else None, kind=case["kind"], alpha=case["alpha"], eps=1e-5)
        else:
            y, h = _plain_norms(st)
        return {"y": y} if h is None else {"y": y, "h": h}
    if own:
        lam = ops.diff_lambda(st["lq1"], st["lk1"], st["lq2"], st["lk2"], st["init"])
        o = ops.diff_attention(st["q"], st["k"], st["v"], lam, st["cu_q"], st["cu_k"], case["B"], case["heads"], case["kv_heads"], st["Lq"],
                               case["L"], case["causal"], key_ids=st["ids"], norm_w=st["w"], out_scale=1.0 - st["init"], eps=1e-5)
    else:
        o = _plain_attention(st)
    return {"o": o}


_LEAVES = {"rotary": ("q", "k"), "norms": ("x", "f", "z", "s", "pw", "pb", "nw", "nb"),
           "attention": ("q", "k", "v", "lq1", "lk1", "lq2", "lk2", "w")}
_GRADS = {"q": "gq", "k": "gk", "y": "gx", "h": "gh", "o": "gy"}


def run(state: dict) -> tp.Dict[str, torch.Tensor]:
    case = state["case"]
    if not case["train"]:
        with torch.no_grad():
            return _forward(state)
    out = _forward(state)
    names = [n for n in _LEAVES[case["op"]] if state[n] is not None]
    grads = torch.autograd.grad(list(out.values()), [state[n] for n in names], [state[_GRADS[n]] for n in out])
    return {**{n: t.detach() for n, t in out.items()}, **{"d_" + n: t for n, t in zip(names, grads)}}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------------------
def _exact_rotary(st: dict) -> tp.Dict[str, torch.Tensor]:
    case = st["case"]
    turn = torch.polar(torch.full_like(st["freq"], st["gain"])[None].expand(case["rows"], -1).contiguous(),
                       st["pos"].double()[:, None] * st["freq"][None])[:, None]

    def apply(x: torch.Tensor, heads: int, by: torch.Tensor) -> torch.Tensor:
        y = x.detach().double().view(case["rows"], heads, case["hd"]).clone()
        half = case["rot"] // 2
        first = slice(0, case["rot"], 2) if case["interleaved"] else slice(0, half)
        second = slice(1, case["rot"], 2) if case["interleaved"] else slice(half, case["rot"])
        c = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * by
        y[..., first], y[..., second] = c.real, c.imag
        return y.reshape(case["rows"], -1)

    out = {"q": apply(st["q"], case["heads"], turn), "k": apply(st["k"], case["kv_heads"], turn)}
    if case["train"]:
        out["d_q"], out["d_k"] = apply(st["gq"], case["heads"], turn.conj()), apply(st["gk"], case["kv_heads"], turn.conj())
    return out


def _exact_norms(st: dict) -> tp.Dict[str, torch.Tensor]:
    case = st["case"]
    up = lambda t: None if t is None else t.detach().double()      # noqa: E731
    x, f, z, s, pw, pb, nw, nb = (up(st[n]) for n in _LEAVES["norms"])
    layer = case["kind"] == "layer"

    def unit(t: torch.Tensor) -> tp.Tuple[torch.Tensor, torch.Tensor]:
        c = t - t.mean(1, keepdim=True) if layer else t
        r = 1.0 / torch.sqrt((c ** 2).mean(1, keepdim=True) + 1e-5)
        return c * r, r

    def unit_back(g: torch.Tensor, u: torch.Tensor, r: torch.Tensor) -> torch.Tensor:
        g = g - u * (g * u).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if layer else 0.0)
        return g * r

    if case["post"]:
        u, ru = unit(f)
        n = u * pw + (pb if pb is not None else 0.0)
    else:
        n = f
    gate = torch.sigmoid(z) if z is not None else torch.ones((), dtype=torch.float64, device=DEV)
    scale = s if s is not None else torch.ones((), dtype=torch.float64, device=DEV)
    y = case["alpha"] * x + scale * gate * n
    out = {"y": y}
    if case["pre"]:
        t, rt = unit(y)
        out["h"] = t * nw + (nb if nb is not None else 0.0)
    if not case["train"]:
        return out
    gy = up(st["gx"])
    if case["pre"]:
        gh = up(st["gh"])
        gy = gy + unit_back(gh * nw, t, rt)
    out["d_x"] = case["alpha"] * gy
    gn = gy * scale * gate
    out["d_f"] = unit_back(gn * pw, u, ru) if case["post"] else gn
    if z is not None:
        out["d_z"] = gy * scale * n * gate * (1.0 - gate)
    if s is not None:
        out["d_s"] = (gy * gate * n).sum(0)
    if case["post"]:
        out["d_pw"] = (gn * u).sum(0)
        if pb is not None:
            out["d_pb"] = gn.sum(0)
    if case["pre"]:
        out["d_nw"] = (gh * t).sum(0)
        if nb is not None:
            out["d_nb"] = gh.sum(0)
    return out


def _exact_attention(st: dict) -> tp.Dict[str, torch.Tensor]:
    """Session by session and head by head, the gradients from their formulas."""
    case = st["case"]
    B, L, H, Hk, hd = case["B"], case["L"], case["heads"], case["kv_heads"], case["hd"]
    q, k, v, q1, k1, q2, k2, w = (st[n].detach().double() for n in _LEAVES["attention"])
    e1, e2 = torch.exp((q1 * k1).sum(1)), torch.exp((q2 * k2).sum(1))
    lam = e1 - e2 + st["init"]
    c, train = 1.0 - st["init"], case["train"]
    cu_k = [L * b for b in range(B + 1)] if st["cu_k"] is None else st["cu_k"].tolist()
    cu_q = [st["Lq"] * b for b in range(B + 1)] if st["cu_q"] is None else st["cu_q"].tolist()
    out = torch.zeros_like(q)
    dq, dk, dv, dw = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(w)
    dlam = torch.zeros_like(lam)
    # sessions of one length go together: [sessions, heads] at a time
    groups: tp.Dict[tp.Tuple[int, int], tp.List[int]] = {}
    for b in range(B):
        groups.setdefault((cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]), []).append(b)
    share = torch.arange(H, device=DEV) // (H // Hk)
    for (n, m), members in groups.items():
        step = max(1, int(2e8 // max(1, n * m * H)))
        for i in range(0, len(members), step):
            some = members[i:i + step]
            rq = torch.stack([torch.arange(cu_q[b], cu_q[b] + n) for b in some]).to(DEV)
            rk = torch.stack([torch.arange(cu_k[b], cu_k[b] + m) for b in some]).to(DEV)
            Q = q[rq].view(len(some), n, H, 2, hd).permute(3, 0, 2, 1, 4)
            K = k[rk].view(len(some), m, Hk, 2, hd)[:, :, share].permute(3, 0, 2, 1, 4)
            V = v[rk].view(len(some), m, Hk, 2 * hd)[:, :, share].transpose(1, 2)
            hide = torch.zeros(len(some), 1, n, m, dtype=torch.bool, device=DEV)
            if st["ids"] is not None:
                hide = hide | (st["ids"][rk] == 0)[:, None, None, :]
            if case["causal"]:
                hide = hide | torch.ones(n, m, dtype=torch.bool, device=DEV).triu(m - n + 1)
            A = []
            for j in (0, 1):
                t = (Q[j] @ K[j].transpose(-1, -2)) / math.sqrt(hd)
                t = torch.softmax(t.masked_fill(hide, -1e300), -1).masked_fill(hide, 0.0)
                A.append(t)
            lamh = lam[:, None, None]
            D = A[0] - lamh * A[1]
            o = D @ V
            r = 1.0 / torch.sqrt((o ** 2).mean(-1, keepdim=True) + 1e-5)
            u = o * r
            put = lambda t: t.transpose(1, 2).reshape(len(some), n, -1)      # noqa: E731
            out[rq] = put(u * w * c)
            if not train:
                continue
            g = st["gy"].double()[rq].view(len(some), n, H, 2 * hd).transpose(1, 2)
            dw += (c * g * u).sum((0, 1, 2))
            gu = g * w * c
            go = r * (gu - u * (gu * u).mean(-1, keepdim=True))
            G = go @ V.transpose(-1, -2)
            dV = D.transpose(-1, -2) @ go
            dK = []
            for j, sign in ((0, 1.0), (1, -lamh)):
                delta = (A[j] * G).sum(-1, keepdim=True)
                if j == 1:
                    dlam -= delta.sum((0, 2, 3))
                dS = sign * A[j] * (G - delta) / math.sqrt(hd)
                dq.view(-1, H, 2, hd)[rq.reshape(-1), :, j] = (dS @ K[j]).transpose(1, 2).reshape(-1, H, hd)
                dK.append(dS.transpose(-1, -2) @ Q[j])
            dK2 = torch.stack(dK, 3).view(len(some), Hk, H // Hk, m, 2, hd).sum(2)      # [b, Hk, m, 2, hd]
            dk[rk] = dK2.transpose(1, 2).reshape(len(some), m, -1)
            dv[rk] = dV.view(len(some), Hk, H // Hk, m, 2 * hd).sum(2).transpose(1, 2).reshape(len(some), m, -1)
    res = {"o": out}
    if train:
        a1, a2 = (dlam * e1)[:, None], (dlam * e2)[:, None]
        res.update(d_q=dq, d_k=dk, d_v=dv, d_lq1=a1 * k1, d_lk1=a1 * q1, d_lq2=-a2 * k2, d_lk2=-a2 * q2, d_w=dw)
    return res


def exact(case: dict, seed: int) -> tp.Dict[str, torch.Tensor]:
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "norms": _exact_norms, "attention": _exact_attention}[case["op"]](st)
