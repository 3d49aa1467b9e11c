"""Differential attention where rows are exactly zero: queries without a gradient (rows without a target, padded rows), zero values, queries and keys,
next to rows of ordinary and of very small size.  A zero row has no size that its neighbours could be measured against.

Tolerance, per tensor, in the 2-norm.  An operand held as two halves is off by 2 u (u = 2^-24), the term that a product of them drops by 4 u more: a
product's factors and the term, 8 u.  What such roundings can do to a result depends on the inputs (a row whose two maps nearly cancel is divided by
the little that is left), so the same formulas are run in 64 bits with every logit, probability, dO v^T and both maps' outputs moved by 8 u, up or
down at random, and q, k, v, dy by 2 u, four times; a result may be off by three times the root mean square of what that moves it (roundings of one
tensor in a row are not independent of each other), three times what the formulas in fp32 tensors are off by (sums; the norm), and 16 u of its own size
(two products follow each other on every path)."""
import math

import pytest
import torch

from test_diff_layers_gpu import STACK_K, _batch, _near, _plain as _plain_stack, _stack

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LENS = [70, 33, 5, 129]
NAMES = ("y", "dq", "dk", "dv", "dlam", "dw")


def _plain(ins, gy, lens_q, lens_k, H, Hkv, causal, c, eps, dtype, noise=None):
    """{name: tensor} of the formulas in `dtype`, session by session, gradients by autograd.  noise: the generator of the roundings."""
    def off(t, by):
        return t if noise is None else t * (1.0 + by * U * (2.0 * torch.randint(0, 2, t.shape, generator=noise) - 1.0))

    q, k, v, lam, w = (None if t is None else t.detach().clone().to(dtype) for t in ins)
    q, k, v, lam, w = (None if t is None else t.requires_grad_() for t in (off(q, 2), off(k, 2), off(v, 2), lam, w))
    hd, share, out, a, b = q.shape[1] // (2 * H), torch.arange(H) // (H // Hkv), [], 0, 0
    for nq, nk in zip(lens_q, lens_k):
        Q = q[a:a + nq].view(nq, H, 2, hd).permute(1, 2, 0, 3)
        K = k[b:b + nk].view(nk, Hkv, 2, hd).permute(1, 2, 0, 3)[share]
        V = v[b:b + nk].view(nk, Hkv, 2 * hd).transpose(0, 1)[share]
        s = off(Q @ K.transpose(-1, -2) / math.sqrt(hd), 8)
        if causal:
            s = s.masked_fill(torch.ones(nq, nk, dtype=torch.bool).triu(nk - nq + 1), -math.inf)
        A = torch.softmax(s, -1)
        if noise is None:
            o = (A[:, 0] - lam[:, None, None] * A[:, 1]) @ V
        else:
            if gy is not None:
                A.register_hook(lambda t: off(t, 8))
            m = off(off(A, 8) @ V[:, None], 8)
            o = m[:, 0] - lam[:, None, None] * m[:, 1]
        if w is not None:
            o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + eps) * w
        out.append((c * o).transpose(0, 1).reshape(nq, -1))
        a, b = a + nq, b + nk
    y = torch.cat(out)
    got = {"y": y.detach()}
    if gy is not None:
        leaves = [(n, t) for n, t in zip(NAMES[1:], (q, k, v, lam, w)) if t is not None]
        got.update(zip([n for n, _ in leaves], torch.autograd.grad(y, [t for _, t in leaves], off(gy.to(dtype), 2))))
    return got


def _check(ins, gy, lens_q, lens_k, H, Hkv, causal, c=0.64, eps=1e-5):
    from rectools_amd import ops

    cu = lambda lens: torch.tensor([0] + lens).cumsum(0).cuda()      # noqa: E731
    q, k, v, lam, w = (None if t is None else t.cuda().requires_grad_(gy is not None) for t in ins)
    y = ops.diff_attention(q, k, v, lam, cu(lens_q), cu(lens_k), len(lens_q), H, Hkv, max(lens_q), max(lens_k), causal, norm_w=w, out_scale=c, eps=eps)
    got = {"y": y.detach()}
    if gy is not None:
        leaves = [(n, t) for n, t in zip(NAMES[1:], (q, k, v, lam, w)) if t is not None]
        got.update(zip([n for n, _ in leaves], torch.autograd.grad(y, [t for _, t in leaves], gy.cuda())))
    want, near = (_plain(ins, gy, lens_q, lens_k, H, Hkv, causal, c, eps, t) for t in (torch.float64, torch.float32))
    g = torch.Generator().manual_seed(1)
    moved = [_plain(ins, gy, lens_q, lens_k, H, Hkv, causal, c, eps, torch.float64, g) for _ in range(4)]
    for n, t in got.items():
        rms = math.sqrt(sum(float((m[n] - want[n]).square().sum()) for m in moved) / 4)
        off, plain, size = float((t.cpu().double() - want[n]).norm()), float((near[n].double() - want[n]).norm()), float(want[n].norm())
        assert off <= 3 * rms + 3 * plain + 16 * U * size, f"{n}: off by {off / size:.2e} of its size, fp32 tensors by {plain / size:.2e}, roundings {rms / size:.2e}"
    return got


def _inputs(nq, nk, H, Hkv, hd, norm, seed=0):
    g = torch.Generator().manual_seed(seed + hd)
    q, k, v = (torch.randn(n, h * 2 * hd, generator=g) for n, h in ((nq, H), (nk, Hkv), (nk, Hkv)))
    return [q, k, v, torch.rand(H, generator=g) * 0.8 + 0.1, 1.0 + 0.1 * torch.randn(2 * hd, generator=g) if norm else None], torch.randn(nq, H * 2 * hd, generator=g), g


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e-6, 1e-8])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,hd,norm", [(2, 2, 32, True), (2, 1, 64, False), (1, 1, 20, True)])
def test_queries_without_a_gradient(H, Hkv, hd, norm, causal, size):
    n = sum(LENS)
    ins, gy, g = _inputs(n, n, H, Hkv, hd, norm)
    none = torch.rand(n, generator=g) < 0.85
    none[[3, 80, 105, 200]] = False
    got = _check(ins, torch.where(none[:, None], 0.0, gy * size), LENS, LENS, H, Hkv, causal)
    assert not got["dq"][none.cuda()].any()


@pytest.mark.parametrize("size", [1e4, 1.0, 1e-3, 1e-6, 1e-9])
@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("H,Hkv,hd,norm", [(2, 2, 32, True), (2, 1, 64, False)])
@pytest.mark.parametrize("share", [0.05, 0.5, 0.95])
def test_zero_values(share, H, Hkv, hd, norm, train, size):
    n = sum(LENS)
    ins, gy, g = _inputs(n, n, H, Hkv, hd, norm, seed=1)
    none = torch.rand(n, generator=g) < share
    none[[10, 71, 104, 130]] = True
    none[[0, 70, 103, 108]] = False
    ins[2] = torch.where(none[:, None], 0.0, ins[2] * size)
    _check(ins, gy if train else None, LENS, LENS, H, Hkv, True)
    _check(ins, gy if train else None, LENS, LENS, H, Hkv, False)


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-6])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("causal", [True, False])
def test_zero_queries_and_keys(causal, which, size):
    """The other operand is as much larger, so that the logits are what they are without the sizes."""
    n = sum(LENS)
    ins, gy, g = _inputs(n, n, 2, 1, 32, True, seed=2)
    none = torch.rand(n, generator=g) < 0.5
    ins[which] = torch.where(none[:, None], 0.0, ins[which] * size)
    ins[1 - which] = ins[1 - which] / size
    _check(ins, gy, LENS, LENS, 2, 1, causal)


@pytest.mark.parametrize("rows", [1, 40])
def test_zero_values_of_split_keys(rows):
    """Few queries and few matrix tiles against long keys."""
    for size in (1.0, 1e-6):
        ins, _, g = _inputs(rows, 3_000, 2, 1, 32, False, seed=3)
        none = torch.rand(3_000, generator=g) < 0.3
        none[1_000:2_000] = True
        ins[2] = torch.where(none[:, None], 0.0, ins[2] * size)
        _check(ins, None, [rows], [3_000], 2, 1, True)


@pytest.mark.parametrize("size", [1.0, 1e-6])
@pytest.mark.parametrize("causal,keypad", [(False, True), (True, False)])
def test_stack_with_few_targets(causal, keypad, size):
    """The upstream gradient is zero but for a few rows, as behind a loss over masked positions."""
    B, L = 4, 70
    layers = _stack()
    ids, x, up = _batch(B, L, 7)
    see = torch.ones(L, L, dtype=torch.bool).tril() if causal else torch.ones(L, L, dtype=torch.bool)
    see = see[None].expand(B, L, L) & ((ids != 0)[:, None, :] if keypad else torch.ones(B, 1, L, dtype=torch.bool))
    at = torch.zeros(B, L, dtype=torch.bool)
    at[0, 5::9], at[1, -1], at[2, 40::8], at[3, -2:] = True, True, True, True
    up = torch.where(at.reshape(-1)[:, None], up * size, 0.0)
    xr = x.double().requires_grad_()
    want, P = _plain_stack(layers, xr, torch.arange(L).repeat(B), see, B, L)
    wg = dict(zip(["x"] + list(P), torch.autograd.grad(want, [xr] + list(P.values()), up.double())))
    xd = x.cuda().requires_grad_()
    params = dict(layers.named_parameters())
    got = torch.autograd.grad(layers(xd, ids.cuda().reshape(-1), B, L, causal, keypad, {}), [xd] + list(params.values()), up.cuda())
    for n, t in zip(["x"] + list(params), got):
        _near(t, wg[n], 4 * STACK_K, n)
