"""Rotary positions, differential attention and the fused norms / gate / residual scale on the GPU against plain implementations in 64 bits
(CPU), at the sizes, layouts and masks where they can go wrong.

Tolerances.  u = 2^-24 is half a step of fp32.  A sum of n products carries at most (n + 1) u of the sum of its terms' magnitudes, whatever
its order.  A split product x y ~ h h' + h l' + l h' adds: x against h + l — h rounds x, at least 2^k, by 2^(k - 11) at most, l rounds that by 2^(k - 23)
at most: 2 u of x; the same for y; the dropped l l': 2^-11 of x times 2^-11 of y: 4 u — 8 u of the product, and its sum has three terms
for one.  (Values below 2^-17 of their row's largest carry 2^-38 of that instead: nothing here.)  The references below return, next to every
result, its MAGNITUDE: the same formula over absolute values.  A result may then be off by k * magnitude, with k counted from the lengths of the
sums that lead to it (`_kappa`)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ops():
    from rectools_amd import ops

    return ops


def _dev():
    return torch.device("cuda:0")


def _close(got, want, mag, k, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - want).abs()
    bad = err > k * mag + 1e-37
    if bad.any():
        i = int((err / (k * mag + 1e-37)).argmax())
        raise AssertionError(f"{what}: off by {float(err.flatten()[i]):.3e} at {i}, allowed {float((k * mag).flatten()[i]):.3e} "
                             f"({int(bad.sum())} of {bad.numel()} elements)")


# ---- rotary ------------------------------------------------------------------------------------------------------------------------------
def _rotary_ref(x, pos, freq, heads, interleaved, gain, back=False):
    M, hd, rot = x.shape[0], x.shape[1] // heads, 2 * freq.numel()
    y = x.double().view(M, heads, hd).clone()
    phi = (pos.double()[:, None] * freq[None])[:, None] * (-1.0 if back else 1.0)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a.clone(), b.clone()
    na, nb = gain * (a * phi.cos() - b * phi.sin()), gain * (a * phi.sin() + b * phi.cos())
    mag = y.abs().clone()
    m = gain * (a.abs() + b.abs())
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2], mag[..., 0:rot:2], mag[..., 1:rot:2] = na, nb, m, m
    else:
        y[..., :rot // 2], y[..., rot // 2:rot], mag[..., :rot // 2], mag[..., rot // 2:rot] = na, nb, m, m
    return y.reshape(M, -1), mag.reshape(M, -1)


# sine and cosine of the reduced angle: 2 u for the rounding of the fraction (|2 pi frac| <= pi: pi u absolute), 4 u for the library function's
# steps, u for the gain, 2 u for the product and the sum of two of them
ROT_K = 12 * U


@pytest.mark.parametrize("M,heads,kv,hd,rot,inter,far", [
    (1, 1, 1, 2, 2, False, 0), (1, 8, 8, 32, 32, False, 0), (3, 2, 1, 9, 6, True, 0), (65, 4, 2, 25, 24, False, 7), (200, 4, 4, 64, 32, True, 3_000_000_000),
    (777, 8, 2, 64, 64, False, 1_000_000), (40_000, 8, 2, 128, 64, False, 0), (64, 1, 1, 8, 8, True, -500), (33, 3, 1, 600, 600, False, 12), (5, 2, 2, 12, 4, True, 0)])
def test_rotary(M, heads, kv, hd, rot, inter, far):
    ops = _ops()
    g = torch.Generator().manual_seed(M + hd)
    q, k = torch.randn(M, heads * hd, generator=g), torch.randn(M, kv * hd, generator=g)
    pos = torch.randint(0, 1000, (M,), generator=g) + far
    freq, gain = ops.rotary_frequencies(rot, scaling="parts", factor=4.0)
    dev = _dev()
    qd, kd = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()
    q2, k2 = ops.rotary_qk(qd, kd, pos.to(dev), freq.to(dev), heads, kv, inter, gain)
    for got, x, n, what in ((q2, q, heads, "q"), (k2, k, kv, "k")):
        _close(got, *_rotary_ref(x, pos, freq, n, inter, gain), ROT_K, what)
    gq, gk = torch.randn(M, heads * hd, generator=g), torch.randn(M, kv * hd, generator=g)
    dq, dk = torch.autograd.grad((q2, k2), (qd, kd), (gq.to(dev), gk.to(dev)))
    for got, x, n, what in ((dq, gq, heads, "dq"), (dk, gk, kv, "dk")):
        _close(got, *_rotary_ref(x, pos, freq, n, inter, gain, back=True), ROT_K, what)
    only = ops.rotary(qd.detach(), pos.to(dev), freq.to(dev), heads, inter, gain)
    assert torch.equal(only, q2.detach())


def test_rotary_reads_column_blocks_in_place_and_one_gradient_alone():
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(50, 3 * 64, generator=g)
    freq, _ = ops.rotary_frequencies(16)
    pos = torch.arange(50)
    d = qkv.to(dev).requires_grad_()
    q2, k2 = ops.rotary_qk(d[:, :64], d[:, 64:128], pos.to(dev), freq.to(dev), 4, 4)
    _close(q2, *_rotary_ref(qkv[:, :64].contiguous(), pos, freq, 4, False, 1.0), ROT_K, "q block")
    _close(k2, *_rotary_ref(qkv[:, 64:128].contiguous(), pos, freq, 4, False, 1.0), ROT_K, "k block")
    up = torch.randn(50, 64, generator=g)
    (dx,) = torch.autograd.grad(k2, d, up.to(dev))      # q2 has no gradient
    want, mag = _rotary_ref(up, pos, freq, 4, False, 1.0, back=True)
    _close(dx[:, 64:128], want, mag, ROT_K, "k block gradient")
    assert not dx[:, :64].any() and not dx[:, 128:].any()
    # odd row strides and offsets: no vector loads
    w = torch.randn(50, 67, generator=g)
    y = ops.rotary(w.to(dev)[:, 1:65], pos.to(dev), freq.to(dev), 4)
    _close(y, *_rotary_ref(w[:, 1:65].contiguous(), pos, freq, 4, False, 1.0), ROT_K, "odd stride")
    e = ops.rotary(torch.randn(0, 64, device=dev), torch.zeros(0, dtype=torch.int64, device=dev), freq.to(dev), 4)
    assert e.shape == (0, 64)


def test_rotary_refusals():
    ops, dev = _ops(), _dev()
    x, pos = torch.randn(4, 32, device=dev), torch.arange(4, device=dev)
    freq = ops.rotary_frequencies(8, device=dev)[0]
    for bad in (lambda: ops.rotary(x, pos[:3], freq, 4), lambda: ops.rotary(x, pos.int(), freq, 4), lambda: ops.rotary(x, pos, freq.float(), 4),
                lambda: ops.rotary(x, pos, freq, 3), lambda: ops.rotary(x, pos, freq, 8), lambda: ops.rotary(x, pos, freq, 0), lambda: ops.rotary(x[0], pos, freq, 4),
                lambda: ops.rotary_qk(x, x[:2], pos, freq, 4, 4), lambda: ops.rotary_qk(x, x, pos, freq, 4, 2)):
        with pytest.raises(ValueError):
            bad()
    from rectools_amd._lib import HipLibraryError

    for bad in (lambda: ops.rotary(x.half(), pos, freq, 4), lambda: ops.rotary(x.cpu(), pos, freq, 4)):
        with pytest.raises(HipLibraryError):
            bad()


# ---- differential attention -----------------------------------------------------------------------------------------------------------------
def _attention_ref(q, k, v, lam, lens_q, lens_k, H, Hkv, causal, ids, w, c, eps, gy=None, scale=None):
    """Session by session in 64 bits: results and their magnitudes ({name: (value, magnitude)}), and the largest logit magnitude."""
    q, k, v, lam = q.double(), k.double(), v.double(), lam.double()
    hd = q.shape[1] // (2 * H)
    sc = 1.0 / math.sqrt(hd) if scale is None else scale
    names = {"y": q, "dq": q, "dk": k, "dv": v, "dlam": lam}
    out = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in names.items()}
    dw = torch.zeros(2 * hd, dtype=torch.float64), torch.zeros(2 * hd, dtype=torch.float64)
    top, rho, qs, ks = 0.0, 1.0, 0, 0
    for nq, nk in zip(lens_q, lens_k):
        for h in range(H):
            hk = h // (H // Hkv)
            cq, cv = slice(h * 2 * hd, (h + 1) * 2 * hd), slice(hk * 2 * hd, (hk + 1) * 2 * hd)
            Q, K, V = q[qs:qs + nq, cq].reshape(nq, 2, hd), k[ks:ks + nk, cv].reshape(nk, 2, hd), v[ks:ks + nk, cv]
            see = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                see = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)
            if ids is not None:
                see = see & (ids[ks:ks + nk] != 0)[None]
                live = (ids[ks:ks + nk] != 0)[:, None]
                K, V = torch.where(live[..., None], K, 0.0), torch.where(live, V, 0.0)
            A = []
            for m in (0, 1):
                s = (Q[:, m] @ K[:, m].T) * sc
                sm = (Q[:, m].abs() @ K[:, m].abs().T) * sc
                if see.any():
                    top = max(top, float(sm[see].max()))
                s = s.masked_fill(~see, -math.inf)
                e = torch.exp(s - torch.where(see.any(1), s.amax(1) if nk else torch.zeros(nq, dtype=torch.float64), 0.0)[:, None]).masked_fill(~see, 0.0)
                t = e.sum(1, keepdim=True)
                A.append(e / torch.where(t > 0, t, 1.0))
            o, om = (A[0] - lam[h] * A[1]) @ V, (A[0] + lam[h].abs() * A[1]) @ V.abs()
            if w is not None:
                r = 1.0 / torch.sqrt((o * o).mean(1, keepdim=True) + eps)
                ow = w.double()
            else:
                r, ow = torch.ones(nq, 1, dtype=torch.float64), torch.ones(2 * hd, dtype=torch.float64)
            amp = 1.0 + r * (om * om).mean(1, keepdim=True).sqrt() if w is not None else torch.ones(nq, 1, dtype=torch.float64)
            rho = max(rho, float(amp.max())) if nq else rho
            out["y"][0][qs:qs + nq, cq], out["y"][1][qs:qs + nq, cq] = c * ow * o * r, abs(c) * ow.abs() * r * (om + o.abs() * amp)
            if gy is None:
                continue
            G = gy.double()[qs:qs + nq, cq]
            if w is not None:
                uu, um, gu = o * r, om * r, c * ow * G
                do = r * (gu - uu * (gu * uu).mean(1, keepdim=True))
                dom = r * (gu.abs() + um * (gu.abs() * um).mean(1, keepdim=True)) * amp
                dw[0].add_((c * G * uu).sum(0))
                dw[1].add_((abs(c) * G.abs() * um * amp).sum(0))
            else:
                do, dom = c * G, abs(c) * G.abs()
            P, Pm = do @ V.T, dom @ V.abs().T
            out["dv"][0][ks:ks + nk, cv] += (A[0] - lam[h] * A[1]).T @ do
            out["dv"][1][ks:ks + nk, cv] += (A[0] + lam[h].abs() * A[1]).T @ dom
            for m, sg in ((0, 1.0), (1, -lam[h])):
                dl, dlm = (A[m] * P).sum(1, keepdim=True), (A[m] * Pm).sum(1, keepdim=True)
                dS, dSm = sg * A[m] * (P - dl) * sc, abs(sg) * A[m] * (Pm + dlm) * sc
                cm = slice(h * 2 * hd + m * hd, h * 2 * hd + (m + 1) * hd)
                ck = slice(hk * 2 * hd + m * hd, hk * 2 * hd + (m + 1) * hd)
                out["dq"][0][qs:qs + nq, cm], out["dq"][1][qs:qs + nq, cm] = dS @ K[:, m], dSm @ K[:, m].abs()
                out["dk"][0][ks:ks + nk, ck] += dS.T @ Q[:, m]
                out["dk"][1][ks:ks + nk, ck] += dSm.T @ Q[:, m].abs()
                if m == 1:
                    out["dlam"][0][h] -= dl.sum()
                    out["dlam"][1][h] += dlm.sum()
        qs, ks = qs + nq, ks + nk
    out["dw"] = dw
    return out, top, rho


def _kappa(hd, n, top, rho):
    """A logit of magnitude `top` is off by d = (3 hd + 12) u top (its sum of 3 hd terms, the split, the scales), a probability by 2 d + 8 u relative (the
    exponential, its argument's rounding against the maximum); products over n keys add (3 n + 9) u and the row sum n u; a gradient passes the
    probability twice and its own sums (3 * 2 hd and 2 hd of delta); the statistics of the norm amplify what o is off by through rho (counted in the
    magnitudes of o, once more here)."""
    d = (3 * hd + 12) * U * top
    return (2 * d + 8 * U) * 2 + (4 * n + 8 * hd + 32) * U * (1.0 + 0.25 * rho)


def _cu(lens):
    return torch.tensor([0] + lens).cumsum(0)


def _attention_case(lens_q, lens_k, H, Hkv, hd, causal, ids=None, w=True, packed_q=True, packed_k=True, train=True, seed=0, tail=0, spread=1.0, Lq=None,
                    Lk=None, scale=None, sizes=None):
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(seed + hd * 7 + H)
    B, Nq, Nk = len(lens_q), sum(lens_q), sum(lens_k)
    q, k, v = (torch.randn(n, c * 2 * hd, generator=g) * s for n, c, s in ((Nq, H, spread), (Nk, Hkv, 1.0), (Nk, Hkv, 1.0)))
    if sizes is not None:      # every row times a size of its own
        q, k, v = (t * f[:, None].float() for t, f in zip((q, k, v), sizes(g, Nq, Nk)))
    lam, wt = torch.rand(H, generator=g) * 0.8 + 0.1, (1.0 + 0.1 * torch.randn(2 * hd, generator=g)) if w else None
    gy = torch.randn(Nq, H * 2 * hd, generator=g)
    c, eps = 0.64, 1e-5
    want, top, rho = _attention_ref(q, k, v, lam, lens_q, lens_k, H, Hkv, causal, ids, wt, c, eps, gy if train else None, scale)
    junk = lambda t: torch.cat([t, torch.full((tail, t.shape[1]), float("nan"))]) if tail else t      # noqa: E731
    qd, kd, vd = (junk(t).to(dev).requires_grad_(train) for t in (q, k, v))
    lamd, wd = lam.to(dev).requires_grad_(train), None if wt is None else wt.to(dev).requires_grad_(train)
    idd = None if ids is None else torch.cat([ids, torch.ones(tail, dtype=torch.int64)]).to(dev)
    y = ops.diff_attention(qd, kd, vd, lamd, _cu(lens_q).to(dev) if packed_q else None, _cu(lens_k).to(dev) if packed_k else None, B, H, Hkv,
                           Lq if Lq is not None else (max(lens_q) if B else 0), Lk if Lk is not None else (max(lens_k) if B else 0), causal, key_ids=idd,
                           norm_w=wd, out_scale=c, eps=eps, scale=scale)
    k_ = _kappa(hd, max(lens_k + [1]), top, rho)
    assert not y[Nq:].any()      # rows behind the last session
    _close(y[:Nq], *want["y"], k_, "y")
    if not train:
        return y
    leaves = {"dq": qd, "dk": kd, "dv": vd, "dlam": lamd}
    if wd is not None:
        leaves["dw"] = wd
    up = torch.cat([gy, torch.full((tail, gy.shape[1]), float("nan"))]) if tail else gy
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), up.to(dev))))
    n_sum = max(lens_k + lens_q + [1]) * (H // Hkv)
    for n, t in grads.items():
        rows = {"dq": Nq, "dk": Nk, "dv": Nk}.get(n)
        if rows is not None:
            assert not t[rows:].any(), n
            t = t[:rows]
        total = n_sum if n in ("dk", "dv", "dq") else 64      # (sums over all rows are held in 64 bits)
        _close(t, *want[n], _kappa(hd, max(max(lens_k + [1]), total), top, rho), n)
    return y


@pytest.mark.parametrize("hd", [1, 4, 9, 16, 25, 32, 33, 48, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_head_sizes(hd, causal):
    _attention_case([1, 31, 70, 0, 129], [1, 31, 70, 0, 129], 2, 2, hd, causal)


@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 63, 64, 65, 200, 333])
def test_attention_lengths(L):
    _attention_case([L, max(1, L - 1)], [L, max(1, L - 1)], 1, 1, 32, True, seed=L)


@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (6, 1), (8, 8), (3, 1)])
@pytest.mark.parametrize("hd", [32, 64, 20])
def test_attention_shared_heads(H, Hkv, hd):
    _attention_case([40, 97], [40, 97], H, Hkv, hd, True)


@pytest.mark.parametrize("lens_q,lens_k", [([1, 1, 1], [1, 70, 300]), ([5, 3, 1], [5, 64, 129]), ([70, 10], [200, 10]), ([64, 3], [20, 1]), ([3, 0, 2], [0, 9, 40])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("train", [True, False])
def test_attention_queries_and_keys_of_different_lengths(lens_q, lens_k, causal, train):
    """The last query meets the last key; with more queries than keys the first ones see nothing, with no keys none does."""
    _attention_case(lens_q, lens_k, 4, 2, 32, causal, train=train)


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd", [25, 32, 64])
def test_attention_padded_windows_with_masked_keys(hd, causal, train):
    L, B = 70, 4
    ids = torch.ones(B, L, dtype=torch.int64)
    ids[0, :69] = 0                       # one key
    ids[1, :] = 0                         # none: every row is empty
    ids[2, 3::2] = 0                      # holes
    y = _attention_case([L] * B, [L] * B, 2, 1, hd, causal, ids=ids.reshape(-1), packed_q=False, packed_k=False, train=train)
    assert not y[L:2 * L].any()


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("q_rows", [1, 70])
def test_attention_masked_rows_may_hold_anything(train, q_rows):
    """NaN and infinities in masked keys and values reach nothing, their gradients are zero."""
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(3)
    L, H, hd = 70, 2, 32
    ids = torch.ones(L, dtype=torch.int64)
    ids[:9] = 0
    ids[40] = 0
    q, k, v = torch.randn(q_rows, H * 64, generator=g), torch.randn(L, H * 64, generator=g), torch.randn(L, H * 64, generator=g)
    res = []
    for fill in (0.0, math.nan, math.inf):
        k2, v2 = (torch.where(ids[:, None] != 0, t, fill).to(dev).requires_grad_(train) for t in (k, v))
        y = ops.diff_attention(q.to(dev), k2, v2, torch.full((H,), 0.4, device=dev), None, None, 1, H, H, q_rows, L, True, key_ids=ids.to(dev))
        res.append([y.detach()] + (list(torch.autograd.grad(y.sum(), (k2, v2))) if train else []))
    for r in res[1:]:
        for a, b in zip(res[0], r):
            assert torch.equal(a, b)
    if train:
        assert not res[0][1][:9].any() and not res[0][2][40].any()


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("q_one", [True, False])
def test_attention_rows_behind_the_last_session(train, q_one):
    lens = [33, 5]
    if q_one:
        _attention_case([1, 1], lens, 2, 2, 32, True, train=train, tail=3)
    else:
        _attention_case(lens, lens, 2, 2, 32, True, train=train, tail=70)


@pytest.mark.parametrize("train", [True, False])
def test_attention_sessions_longer_than_expected(train):
    _attention_case([150, 20], [150, 20], 2, 2, 32, True, train=train, Lq=64, Lk=64)
    _attention_case([9, 2], [150, 20], 2, 2, 32, True, train=train, Lq=1, Lk=40)


@pytest.mark.parametrize("rows,keys", [(1, 5_000), (2, 9_001), (40, 6_000)])
@pytest.mark.parametrize("hd", [32, 64, 17])
def test_attention_split_keys(rows, keys, hd):
    """Few rows against many keys: the keys are split over workgroups and joined."""
    _attention_case([rows], [keys], 4, 2, hd, True, train=False)
    _attention_case([rows, 1], [keys, 3], 2, 1, hd, False, train=False)


@pytest.mark.parametrize("hd", [4, 32, 64])
@pytest.mark.parametrize("H,Hkv", [(2, 2), (4, 2)])
def test_attention_rows_of_one_key_have_no_gradient(hd, H, Hkv):
    """One visible key: its weight is 1 whatever the logits are, dS is exactly zero.  First rows of causal sessions, sessions of one row, one key left
    by the mask."""
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(hd)
    lens = [1, 5, 40, 1]
    cu = _cu(lens).to(dev)
    q, k, v = (torch.randn(47, n * 2 * hd, generator=g).to(dev).requires_grad_() for n in (H, Hkv, Hkv))
    lam, w = torch.full((H,), 0.4, device=dev), torch.rand(2 * hd, generator=g).to(dev) + 0.5
    gy = torch.randn(47, H * 2 * hd, generator=g).to(dev)
    y = ops.diff_attention(q, k, v, lam, cu, cu, 4, H, Hkv, 40, 40, True, norm_w=w)
    dq, dk, _ = torch.autograd.grad(y, (q, k, v), gy)
    assert not dq[[0, 1, 6, 46]].any() and dq[[2, 7, 45]].any(1).all() and not dk[[0, 46]].any()
    ids = torch.zeros(47, dtype=torch.int64)
    ids[[9, 46]] = 1
    y = ops.diff_attention(q, k, v, lam, cu, cu, 4, H, Hkv, 40, 40, False, key_ids=ids.to(dev), norm_w=w)
    dq, dk, _ = torch.autograd.grad(y, (q, k, v), gy)
    assert not dq[46].any() and not dk[46].any() and not dq[:6].any()      # (the 40 rows' session is longer than a chunk: rounding)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_short_sessions_with_one_heavy_key(H, Hkv, causal):
    """Nearly all of the weight on one key h: dS_j = p_j (G_j - sum p G) cancels there to sum over the others of p_j (G_h - G_j), and the gradient of
    q is held to the size of that."""
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(5)
    hd, lens = 32, [2, 3, 9, 30]
    n, sc = sum(lens), 1.0 / math.sqrt(hd)
    q, k, v = (torch.randn(n, c * 2 * hd, generator=g) for c in (H, Hkv, Hkv))
    k = k * 0.02
    k[[0, 2, 5, 14]] = 1.0                 # the first key of every session, seen by all of its rows
    q = q * 0.1 + 1.5                      # logits of about 1.5 * 32 / sqrt(32) = 8.5 there, 0 at the others: weights e^-8.5
    lam = torch.full((H,), 0.4)
    gy = torch.randn(n, H * 2 * hd, generator=g)
    want, top, _ = _attention_ref(q, k, v, lam, lens, lens, H, Hkv, causal, None, None, 1.0, 1e-5, gy)
    qd, kd, vd = (t.to(dev).requires_grad_() for t in (q, k, v))
    cu = _cu(lens).to(dev)
    y = ops.diff_attention(qd, kd, vd, lam.to(dev), cu, cu, 4, H, Hkv, 30, 30, causal)
    dq = torch.autograd.grad(y, qd, gy.to(dev))[0].cpu().double()
    # a weight is off by 2 d + 8 u relative (d: its logit), G by (3 * 2 hd + 12) u of |dO| |v| (no norm: dO = dy), the mean over the keys and the product
    # with k by (4 * 32 + 16) u: all of them of terms p_j (|G_j| + |G_h|) (|k_j| + |k_h|), j not h
    k_ = 2 * (2 * (3 * hd + 12) * U * top + 8 * U) + (6 * hd + 12 + 4 * 32 + 16) * U
    at = 0
    for m in lens:
        see = torch.ones(m, m, dtype=torch.bool).tril() if causal else torch.ones(m, m, dtype=torch.bool)
        for h in range(H):
            hk = h // (H // Hkv)
            G = gy[at:at + m, h * 2 * hd:(h + 1) * 2 * hd].double().abs() @ v[at:at + m, hk * 2 * hd:(hk + 1) * 2 * hd].double().abs().T
            for mp in (0, 1):
                c, ck = (slice((2 * x + mp) * hd, (2 * x + mp + 1) * hd) for x in (h, hk))
                K = k[at:at + m, ck].double()
                p = torch.softmax((q[at:at + m, c].double() @ K.T * sc).masked_fill(~see, -math.inf), 1)
                allowed = ((p[:, 1:] * (G[:, 1:] + G[:, :1]))[..., None] * (K[1:].abs() + K[:1].abs())).sum(1) * sc * (1.0 if mp == 0 else 0.4)
                err = (dq[at:at + m, c] - want["dq"][0][at:at + m, c]).abs()
                assert (err <= k_ * allowed).all(), (m, h, mp, float((err / (k_ * allowed + 1e-300)).max()))
        at += m


@pytest.mark.parametrize("hd", [32, 50, 64])
def test_attention_long_causal_sessions(hd):
    """Few long sessions: two halves of the keys per workgroup; odd counts of chunks, a session without rows, one of a single chunk."""
    _attention_case([600, 289, 0, 33], [600, 289, 0, 33], 2, 1, hd, True, train=True)
    ids = torch.ones(935, dtype=torch.int64)
    ids[::7] = 0
    ids[600:640] = 0
    _attention_case([610, 325], [610, 325], 2, 2, hd, True, ids=ids, train=False)


def test_attention_long_causal_session_in_halves_and_splits():
    _attention_case([2_500], [2_500], 4, 2, 32, True, train=True)


@pytest.mark.parametrize("hd", [32, 50])
@pytest.mark.parametrize("rows", [1, 3, 10])
def test_attention_few_queries_of_sessions_of_different_lengths(hd, rows):
    """Shares of one size: long sessions fill many, short ones one, the rest are empty; sessions without keys and longer than expected among them."""
    lens_k = [9_000, 3, 700, 0, 65, 4_321]
    lens_q = [rows] * 6
    _attention_case(lens_q, lens_k, 2, 2, hd, True, train=False)
    _attention_case(lens_q, lens_k, 2, 1 if rows < 6 else 2, hd, False, train=False, Lk=6_000)
    ids = torch.ones(sum(lens_k), dtype=torch.int64)
    ids[:5_000] = 0
    ids[9_000:9_003] = 0
    _attention_case(lens_q, lens_k, 1, 1, hd, True, train=False, ids=ids)


def test_attention_split_keys_training():
    _attention_case([20], [3_000], 2, 1, 32, True, train=True)


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_attention_flat_and_sharp_maps(spread):
    _attention_case([65, 130], [65, 130], 2, 2, 32, True, spread=spread)


@pytest.mark.parametrize("lens_q,H,Hkv", [([9, 12], 1, 1), ([5, 3], 4, 2), ([4, 1], 3, 1), ([2, 2], 5, 1), ([2, 1], 6, 1), ([1, 1], 8, 1), ([1, 1], 9, 1), ([13], 1, 1)])
@pytest.mark.parametrize("hd", [32, 50])
def test_attention_few_queries_in_one_and_two_passes(lens_q, H, Hkv, hd):
    lens_k = [900 + 70 * i for i in range(len(lens_q))]
    _attention_case(lens_q, lens_k, H, Hkv, hd, True, train=False)
    ids = torch.ones(sum(lens_k), dtype=torch.int64)
    ids[5::3] = 0
    ids[:880] = 0
    _attention_case(lens_q, lens_k, H, Hkv, hd, True, train=False, ids=ids)


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("rows", [1, 80])
def test_attention_rows_of_very_different_sizes(train, rows):
    """Sessions of huge queries and tiny keys, and the other way round, values from 1e-10 to 1e10 next to each other: nothing leaves the range."""
    def sizes(g, nq, nk):
        a = torch.tensor([12.0, -12.0, 3.0]).double()
        at_q, at_k = torch.arange(nq) * 3 // nq, torch.arange(nk) * 3 // nk
        return (10.0 ** (a[at_q] - 4.0 * torch.rand(nq, generator=g)), 10.0 ** (-a[at_k] - 2.0 * torch.rand(nk, generator=g)), 10.0 ** (20.0 * torch.rand(nk, generator=g) - 10.0))
    _attention_case([rows] * 3, [80] * 3, 2, 1, 32, True, w=False, train=train, sizes=sizes)


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_sessions_do_not_see_their_neighbours(rows):
    """A session of NaN between two others, in the same chunk of keys: their rows and gradients keep their bits."""
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(21)
    H, hd, lens = 2, 32, [45, 20, 50]
    cu_q, cu_k = _cu([min(rows, n) for n in lens]).to(dev), _cu(lens).to(dev)
    nq, a, b = int(cu_q[-1]), int(cu_q[1]), int(cu_q[2])
    q, k, v, gy = (torch.randn(n, H * 2 * hd, generator=g).to(dev) for n in (nq, 115, 115, nq))
    lam = torch.full((H,), 0.4, device=dev)
    res = []
    for bad in (False, True):
        ts = [t.clone() for t in (q, k, v)]
        if bad:
            ts[0][a:b], ts[1][45:65], ts[2][45:65] = math.nan, math.inf, math.nan
        with torch.no_grad():
            y0 = ops.diff_attention(*ts, lam, cu_q, cu_k, 3, H, H, max(1, rows), 50, True)
        for t in ts:
            t.requires_grad_()
        y = ops.diff_attention(*ts, lam, cu_q, cu_k, 3, H, H, rows, 50, True)
        res.append([y0, y.detach(), *torch.autograd.grad(y, ts, gy)])
    for i, (x, z) in enumerate(zip(*res)):
        lo, hi = (a, b) if x.shape[0] == nq and i != 3 and i != 4 else (45, 65)
        assert torch.equal(x[:lo], z[:lo]) and torch.equal(x[hi:], z[hi:]), i


@pytest.mark.parametrize("train", [True, False])
def test_attention_without_norm_and_own_scale(train):
    _attention_case([65, 13], [65, 13], 2, 1, 40, True, w=False, train=train)
    _attention_case([65, 13], [65, 13], 2, 1, 32, True, scale=0.3, train=train)


def test_attention_column_blocks_and_empty_calls():
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(9)
    H, hd, n = 2, 32, 77
    qkv = torch.randn(n, 3 * H * 64, generator=g).to(dev)
    lam = torch.full((H,), 0.3, device=dev)
    cu = torch.tensor([0, 30, n], device=dev)
    c = H * 64
    blocks = [qkv[:, i * c:(i + 1) * c] for i in range(3)]
    a = ops.diff_attention(*blocks, lam, cu, cu, 2, H, H, 47, 47, True)
    b = ops.diff_attention(*[t.contiguous() for t in blocks], lam, cu, cu, 2, H, H, 47, 47, True)
    assert torch.equal(a, b)
    odd = torch.randn(n, 3 * c + 1, generator=g).to(dev)
    blocks = [odd[:, 1 + i * c:1 + (i + 1) * c] for i in range(3)]      # unaligned columns
    a = ops.diff_attention(*blocks, lam, cu, cu, 2, H, H, 47, 47, True)
    b = ops.diff_attention(*[t.contiguous() for t in blocks], lam, cu, cu, 2, H, H, 47, 47, True)
    assert torch.equal(a, b)
    e = torch.zeros(0, c, device=dev)
    z = torch.zeros(1, dtype=torch.int64, device=dev)
    assert ops.diff_attention(e, e, e, lam, z, z, 0, H, H, 0, 0, True).shape == (0, c)
    for train in (False, True):      # no sessions: every row is behind the last one
        r = torch.randn(5, c, generator=g).to(dev).requires_grad_(train)
        y = ops.diff_attention(r, r, r, lam, z, z, 0, H, H, 0, 0, True)
        assert not y.any() and (not train or not torch.autograd.grad(y.sum(), r)[0].any())
    e2 = torch.zeros(0, c, device=dev, requires_grad=True)
    y = ops.diff_attention(e2, e2, e2, lam, z, z, 0, H, H, 0, 0, True)
    (d,) = torch.autograd.grad(y.sum(), e2)
    assert d.shape == (0, c)
    q3 = torch.randn(3, c, generator=g).to(dev).requires_grad_()      # queries without any key
    y = ops.diff_attention(q3, e, e, lam, None, None, 1, H, H, 3, 0, True)
    (d,) = torch.autograd.grad(y.sum(), q3)
    assert not y.any() and not d.any()


def test_attention_same_bits_twice_and_gradient_against_differences():
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(11)
    H, Hkv, hd, lens = 4, 2, 16, [40, 90]
    cu = _cu(lens).to(dev)
    q, k, v = (torch.randn(130, c * 2 * hd, generator=g).to(dev).requires_grad_() for c in (H, Hkv, Hkv))
    lam, w = torch.full((H,), 0.4, device=dev, requires_grad=True), torch.ones(2 * hd, device=dev, requires_grad=True)
    gy = torch.randn(130, H * 2 * hd, generator=g).to(dev)
    leaves = (q, k, v, lam, w)

    def run(*ts):
        return ops.diff_attention(*ts[:4], cu, cu, 2, H, Hkv, 90, 90, True, norm_w=ts[4], out_scale=0.5)

    first = torch.autograd.grad(run(*leaves), leaves, gy)
    y = run(*leaves)
    again = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    again = torch.autograd.grad(y, leaves, gy)      # the same graph's second pass
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for i, t in enumerate(leaves):      # a random direction: central differences of sum(gy * y); h^2 terms ~1e-4, rounding of y ~ 1e-6 / h
        d = torch.randn(t.shape, generator=g).to(dev)
        d = d / d.norm()
        h = 1e-2
        with torch.no_grad():
            up, dn = ([s + (d * h * sg if j == i else 0.0) for j, s in enumerate(leaves)] for sg in (1.0, -1.0))
            fd = float(((run(*up).double() - run(*dn).double()) * gy).sum() / (2 * h))
        an = float((first[i] * d).double().sum())
        assert abs(fd - an) <= 2e-2 * max(1.0, abs(an)), (i, fd, an)


def test_diff_lambda():
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(2)
    for H, hd in ((1, 1), (4, 32), (3, 65), (8, 200), (37, 16)):
        vs = [(torch.randn(H, hd, generator=g) * 0.2) for _ in range(4)]
        ds = [t.to(dev).requires_grad_() for t in vs]
        lam = ops.diff_lambda(*ds, 0.35)
        q1, k1, q2, k2 = (t.double() for t in vs)
        e1, e2 = torch.exp((q1 * k1).sum(1)), torch.exp((q2 * k2).sum(1))
        m1, m2 = (q1 * k1).abs().sum(1), (q2 * k2).abs().sum(1)
        # the exponent is off by (hd + 1) u of its terms' magnitudes; exp, two sums: 6 u
        kk = ((hd + 1) * float(torch.maximum(m1, m2).max()) + 6) * U
        _close(lam, e1 - e2 + 0.35, e1 + e2 + 0.35, kk, "lam")
        up = torch.randn(H, generator=g)
        grads = torch.autograd.grad(lam, ds, up.to(dev))
        for got, e, other, s in zip(grads, (e1, e1, e2, e2), (k1, q1, k2, q2), (1, 1, -1, -1)):
            want = s * (up.double() * e)[:, None] * other
            _close(got, want, want.abs(), kk + 4 * U, "lambda gradient")
    with pytest.raises(ValueError):
        ops.diff_lambda(ds[0], ds[1], ds[2], ds[3][:, :1], 0.1)


def test_attention_refusals():
    ops, dev = _ops(), _dev()
    from rectools_amd._lib import HipLibraryError

    q = torch.randn(6, 2 * 2 * 16, device=dev)
    lam, cu = torch.zeros(2, device=dev), torch.tensor([0, 6], device=dev)
    ok = dict(q=q, k=q, v=q, lam=lam, cu_q=cu, cu_k=cu, B=1, H=2, H_kv=2, Lq=6, Lk=6, causal=True)
    ops.diff_attention(**ok)
    for bad in (dict(B=2), dict(H=3), dict(H_kv=1), dict(H=4, H_kv=3), dict(lam=lam[:1]), dict(cu_q=cu.int()), dict(cu_q=cu.cpu()), dict(cu_k=None, Lk=5),
                dict(cu_q=None, Lq=7), dict(k=q[:5]), dict(v=q[:, :32]), dict(q=q[0]), dict(key_ids=cu), dict(norm_w=torch.ones(16, device=dev)),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=1e-60), dict(scale=math.inf), dict(norm_w=torch.ones(32, device=dev), eps=0.0), dict(Lq=-1)):
        with pytest.raises(ValueError):
            ops.diff_attention(**{**ok, **bad})
    wide = torch.randn(6, 2 * 2 * 65, device=dev)
    with pytest.raises(NotImplementedError):
        ops.diff_attention(**{**ok, "q": wide, "k": wide, "v": wide})
    for bad in (dict(q=q.double()), dict(q=q.cpu()), dict(lam=lam.half())):
        with pytest.raises(HipLibraryError):
            ops.diff_attention(**{**ok, **bad})


def _room(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GiB")


@pytest.mark.parametrize("rows", [1, 20])
def test_offsets_beyond_32_bits(rows):
    """Keys, values and rotated columns as blocks of rows 160 kB apart: more than 2^31 elements from the first to the last."""
    _room(32)
    ops, dev = _ops(), _dev()
    n, ld, c = 60_001, 40_000, 64
    wide = torch.empty(n, ld, device=dev)
    blocks = [wide[:, i:i + c] for i in (0, 20_000, ld - c)]
    dense = [torch.randn(n, c, device=dev) for _ in blocks]
    for b, t in zip(blocks, dense):
        b.copy_(t)
    assert wide.stride(0) * (n - 1) > 2 ** 31
    q, lam = torch.randn(rows, c, device=dev), torch.full((1,), 0.3, device=dev)
    ask = lambda k, v: ops.diff_attention(q, k, v, lam, None, None, 1, 1, 1, rows, n, True)      # noqa: E731
    assert torch.equal(ask(*blocks[:2]), ask(*dense[:2]))
    freq, _ = ops.rotary_frequencies(32, device=dev)
    pos = torch.arange(n, device=dev)
    assert torch.equal(ops.rotary(blocks[2], pos, freq, 1), ops.rotary(dense[2], pos, freq, 1))


def test_large_outputs():
    """More than 2^31 elements in and out: the last rows are those of a small call."""
    _room(80)
    ops, dev = _ops(), _dev()
    x = torch.zeros(270_000, 8192, device=dev)
    x[-3:] = torch.randn(3, 8192, device=dev)
    w = torch.rand(8192, device=dev)

    def run(t):
        t = t.detach().requires_grad_()
        y, h = ops.norm_gate_residual(t, t, post=(w, None), pre=(w, None))
        return (y[-3:].detach(), h[-3:].detach(), torch.autograd.grad(h, t, h.detach())[0][-3:])

    assert all(torch.equal(a, b) for a, b in zip(run(x), run(x[-3:].clone())))
    x = x.view(-1, 1280)
    freq, _ = ops.rotary_frequencies(64, device=dev)
    pos = torch.arange(x.shape[0], device=dev)
    assert torch.equal(ops.rotary(x, pos, freq, 20)[-19:], ops.rotary(x[-19:].clone(), pos[-19:], freq, 20))


def test_broadcast_inputs_and_their_gradients():
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(8)
    n, H, hd = 40, 2, 32
    c = H * 2 * hd
    row, lam1, gy = torch.randn(1, c, generator=g).to(dev), torch.tensor([0.4], device=dev), torch.randn(n, c, generator=g).to(dev)
    k = torch.randn(n, c, generator=g).to(dev)
    freq, _ = ops.rotary_frequencies(16, device=dev)
    w = torch.rand(c, generator=g).to(dev) + 0.5
    pos = torch.arange(n, device=dev)

    def run(r, l1, wide):
        x, lam = (r.expand(n, c), l1.expand(H)) if wide else (r, l1)
        y = ops.diff_attention(ops.rotary(x, pos, freq, 2 * H), k, x, lam, None, None, 1, H, H, n, n, True)
        z, h = ops.norm_gate_residual(x, y, gate=x, post=(w, None), pre=(w, None))
        return (z.detach(), h.detach()) + torch.autograd.grad((z, h), (r, l1), (gy, gy[:1].expand(n, c)))

    a = run(row.clone().requires_grad_(), lam1.clone().requires_grad_(), True)
    b = run(row.repeat(n, 1).requires_grad_(), lam1.repeat(H).requires_grad_(), False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for got, each in zip(a[2:], b[2:]):      # the sum over the copies: n terms
        each = each.cpu().double().reshape(-1, got.shape[-1])
        _close(got.reshape(1, -1), each.sum(0, keepdim=True), each.abs().sum(0, keepdim=True), (each.shape[0] + 1) * U, "broadcast")


# ---- norms, gate, residual scale ---------------------------------------------------------------------------------------------------------
def _norm_ref(x, f, z, s, pw, pb, nw, nb, layer, alpha, eps, gy=None, gh=None, keep=None):
    """{name: (value, magnitude)} in 64 bits."""
    up = lambda t: None if t is None else t.double()      # noqa: E731
    x, f, z, s, pw, pb, nw, nb, gy, gh, keep = map(up, (x, f, z, s, pw, pb, nw, nb, gy, gh, keep))

    def unit(t, tm):      # normalised rows; magnitude: the row's own, and what its mean and deviation carry over
        cen = t - t.mean(1, keepdim=True) if layer else t
        cm = tm + tm.mean(1, keepdim=True) if layer else tm
        r = 1.0 / torch.sqrt((cen ** 2).mean(1, keepdim=True) + eps)
        un = cen * r
        return un, cm * r + un.abs() * (1.0 + (cm * r * un.abs()).mean(1, keepdim=True)), r

    def back(g, gm, un, um, r):
        v = r * (g - un * (g * un).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if layer else 0.0))
        m = r * (gm + um * (gm * um).mean(1, keepdim=True) + (gm.mean(1, keepdim=True) if layer else 0.0)) * (1.0 + (um * um).mean(1, keepdim=True).sqrt())
        return v, m

    if pw is not None:
        u1, u1m, r1 = unit(f, f.abs())
        n, nm = u1 * pw + (0.0 if pb is None else pb), u1m * pw.abs() + (0.0 if pb is None else pb.abs())
    else:
        u1, u1m, r1, n, nm = f, f.abs(), None, f, f.abs()
    one = torch.ones((), dtype=torch.float64)
    gate, sc, kp = one if z is None else torch.sigmoid(z), one if s is None else s, one if keep is None else keep
    y, ym = alpha * x + sc * gate * kp * n, abs(alpha) * x.abs() + sc.abs() * gate * kp * nm
    out = {"y": (y, ym)}
    if nw is not None:
        u2, u2m, r2 = unit(y, ym)
        out["h"] = (u2 * nw + (0.0 if nb is None else nb), u2m * nw.abs() + (0.0 if nb is None else nb.abs()))
    if gy is None and gh is None:
        return out
    g = torch.zeros_like(x) if gy is None else gy
    gm = g.abs()
    if gh is not None:
        b, bm = back(gh * nw, (gh * nw).abs(), u2, u2m, r2)
        g, gm = g + b, gm + bm
        out["dnw"], out["dnb"] = ((gh * u2).sum(0), (gh.abs() * u2m).sum(0)), (gh.sum(0), gh.abs().sum(0))
    out["dx"] = (alpha * g, abs(alpha) * gm)
    gn, gnm = g * sc * gate * kp, gm * sc.abs() * gate * kp
    out["df"] = back(gn * pw, gnm * pw.abs(), u1, u1m, r1) if pw is not None else (gn, gnm)
    out["dz"] = (g * sc * n * kp * gate * (1 - gate), gm * sc.abs() * nm * kp * gate)
    out["ds"] = ((g * gate * n * kp).sum(0), (gm * gate * nm * kp).sum(0))
    out["dpw"], out["dpb"] = ((gn * u1).sum(0), (gnm * u1m).sum(0)), (gn.sum(0), gnm.sum(0))
    return out


def _norm_case(M, d, layer, gate=True, scale=True, post=True, pre=True, alpha=1.0, bias=True, use=("y", "h"), p=0.0, shift=0):
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(M * 31 + d)
    rnd = lambda *sh, s=1.0, m=0.0: torch.randn(*sh, generator=g) * s + m      # noqa: E731
    x, f, z = rnd(M, d, s=2.0), rnd(M, d, s=0.5, m=0.2), rnd(M, d) if gate else None
    s = rnd(d, s=0.2, m=0.5) if scale else None
    pw, nw = rnd(d, s=0.1, m=1.0) if post else None, rnd(d, s=0.1, m=1.0) if pre else None
    pb, nb = rnd(d, s=0.1) if post and layer and bias else None, rnd(d, s=0.1) if pre and layer and bias else None

    def place(t):      # shift: rows that start off the 16-byte grid
        if shift and t.dim() == 2:
            flat = torch.empty(t.numel() + shift, device=dev)[shift:].view(t.shape)
            return flat.copy_(t).requires_grad_()
        return t.to(dev).requires_grad_()

    leaves = {n: place(t) for n, t in dict(x=x, f=f, z=z, s=s, pw=pw, pb=pb, nw=nw, nb=nb).items() if t is not None}
    at = leaves.get
    y, h = ops.norm_gate_residual(at("x"), at("f"), gate=at("z"), post=(at("pw"), at("pb")) if post else None, scale=at("s"),
                                  pre=(at("nw"), at("nb")) if pre else None, kind="layer" if layer else "rms", alpha=alpha, p=p)
    assert (h is None) == (not pre)
    gy = rnd(M, d) if "y" in use else None
    gh = rnd(M, d) if "h" in use and pre else None
    want = _norm_ref(x, f, z, s, pw, pb, nw, nb, layer, alpha, 1e-5, gy, gh)
    k = (3 * d + 40) * U      # two statistics and the sums of their gradients over d columns, sigmoid and the products around it
    _close(y, *want["y"], k, "y")
    if pre:
        _close(h, *want["h"], k, "h")
    outs = [(t, u.to(dev)) for t, u in ((y, gy), (h, gh)) if u is not None]
    grads = torch.autograd.grad([t for t, _ in outs], list(leaves.values()), [u for _, u in outs], allow_unused=True)
    for n, t in zip(leaves, grads):
        if ("d" + n) not in want:
            assert t is None or not t.any(), n
            continue
        _close(t, *want["d" + n], k + (M if n in ("s", "pw", "pb", "nw", "nb") else 0) * U, "d" + n)


@pytest.mark.parametrize("d", [1, 2, 3, 16, 50, 63, 64, 65, 100, 128, 130, 256, 257, 260, 500, 512, 513, 1000, 2048, 2049, 4096, 4100, 8192])
@pytest.mark.parametrize("layer", [True, False])
def test_norm_widths(d, layer):
    _norm_case(37, d, layer)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 4097, 20_001])
def test_norm_row_counts(M):
    _norm_case(M, 50, False)
    _norm_case(M, 64, True)


@pytest.mark.parametrize("gate,scale,post,pre", [(a, b, c, e) for a in (0, 1) for b in (0, 1) for c in (0, 1) for e in (0, 1)])
@pytest.mark.parametrize("layer", [True, False])
def test_norm_parts(gate, scale, post, pre, layer):
    _norm_case(70, 48, layer, bool(gate), bool(scale), bool(post), bool(pre), alpha=1.25)


def test_norm_gradients_of_one_output_no_bias_and_unaligned_rows():
    _norm_case(33, 64, True, use=("y",))
    _norm_case(33, 64, True, use=("h",))
    _norm_case(33, 64, True, bias=False)
    for shift in (1, 2, 3):
        _norm_case(33, 64, False, shift=shift)


def test_norm_constant_and_zero_rows():
    """A constant row has no deviation: LayerNorm gives its bias, the gradients stay finite."""
    ops, dev = _ops(), _dev()
    x = torch.zeros(4, 64, device=dev, requires_grad=True)
    f = torch.full((4, 64), 3.0, device=dev, requires_grad=True)
    w, b = torch.ones(64, device=dev, requires_grad=True), torch.full((64,), 0.5, device=dev, requires_grad=True)
    y, h = ops.norm_gate_residual(x, f, post=(w, b), pre=(w, b), kind="layer")
    assert torch.equal(y, torch.full_like(y, 0.5)) and torch.equal(h, torch.full_like(h, 0.5))
    grads = torch.autograd.grad(h.sum(), (x, f, w, b))
    assert all(torch.isfinite(t).all() for t in grads)
    y, h = ops.norm_gate_residual(x, torch.zeros_like(f), post=(w, None), pre=(w, None), kind="rms")
    assert not y.any() and not h.any()


def test_norm_gate_far_from_zero():
    """The gate's slope sigmoid(z) sigmoid(-z) keeps its relative precision where 1 - sigmoid(z) would have none left, and is zero or finite behind that."""
    ops, dev = _ops(), _dev()
    z = torch.tensor([[0.0, 5.0, -5.0, 12.0, -12.0, 17.0, 40.0, -40.0, 80.0, -80.0, 200.0, -200.0]])
    x = torch.ones_like(z)
    zd = z.to(dev).requires_grad_()
    y, _ = ops.norm_gate_residual(x.to(dev), x.to(dev), gate=zd)
    (dz,) = torch.autograd.grad(y.sum(), zd)
    want = torch.sigmoid(z.double()) * torch.sigmoid(-z.double())
    # e^-|z|: its argument is exact, the function 2 u; the sum, the quotient, three products: u each
    assert ((dz.cpu().double() - want).abs() <= 12 * U * want + 1e-37).all(), dz
    want = 1.0 + torch.sigmoid(z.double())
    assert ((y.detach().cpu().double() - want).abs() <= 8 * U * want).all()


@pytest.mark.parametrize("d", [48, 50, 33])
def test_norm_dropout_is_the_row_kernels_mask(d):
    """The mask is the one `ops.dropout` draws for the same (seed, stream, element), in both directions."""
    ops, dev = _ops(), _dev()
    g = torch.Generator().manual_seed(4)
    M, p = 64, 0.3
    x, f, z = (torch.randn(M, d, generator=g) for _ in range(3))
    gy = torch.randn(M, d, generator=g)
    state = ops.RNG.step, ops.RNG._stream
    keep = ops.dropout(torch.ones(M, d, device=dev), p).cpu()
    ops.RNG.step, ops.RNG._stream = state
    assert 0.1 < float((keep == 0).float().mean()) < 0.5
    xs = [t.to(dev).requires_grad_() for t in (x, f, z)]
    y, _ = ops.norm_gate_residual(xs[0], xs[1], gate=xs[2], p=p)
    want = _norm_ref(x, f, z, None, None, None, None, None, False, 1.0, 1e-5, gy, None, keep)
    _close(y, *want["y"], 20 * U, "y")
    for got, n in zip(torch.autograd.grad(y, xs, gy.to(dev)), ("dx", "df", "dz")):
        _close(got, *want[n], 20 * U, n)


def test_norm_same_bits_twice_and_refusals():
    ops, dev = _ops(), _dev()
    from rectools_amd._lib import HipLibraryError

    x, w = torch.randn(5000, 96, device=dev, requires_grad=True), torch.ones(96, device=dev, requires_grad=True)
    one, two = ([t.clone() for t in torch.autograd.grad(ops.norm_gate_residual(x, x, post=(w, None), pre=(w, None))[1].square().sum(), (x, w))] for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    x, w = x.detach()[:4], w.detach()
    for bad in (dict(kind="batch"), dict(p=1.0), dict(p=-0.1), dict(post=(w, w)), dict(post=(None, None)), dict(scale=w[:5]), dict(gate=x[:2]), dict(f=x[:, :5]), dict(x=x[0])):
        with pytest.raises(ValueError):
            ops.norm_gate_residual(**{**dict(x=x, f=x), **bad})
    with pytest.raises(NotImplementedError):
        ops.norm_gate_residual(torch.zeros(1, 8193, device=dev), torch.zeros(1, 8193, device=dev))
    with pytest.raises(HipLibraryError):
        ops.norm_gate_residual(x.double(), x.double())
    e = torch.zeros(0, 96, device=dev, requires_grad=True)
    wl = torch.ones(96, device=dev, requires_grad=True)
    y, h = ops.norm_gate_residual(e, e, post=(wl, None), pre=(wl, None))
    de, dw = torch.autograd.grad(y.sum() + h.sum(), (e, wl))
    assert de.shape == (0, 96) and not dw.any()
