"""The gradient of differential attention's lam over rows that see one key.

Both maps' outputs are that key's values v there: o = (1 - lam) v, dO = r (g - u mean(g u)) with u = o r, r = 1 / sqrt(mean(o^2) + eps), g = c w dy, and the
row's share of dlam is -dO . v = -r (g . v) (1 - mean(o^2) r^2) = -r^3 eps (g . v): about 1e-5 of its terms, all the rest cancels.

Tolerance, u = 2^-24: a saved output is off from v by 14 u (2 for the values' halves, 8 for a product of them, 4 for the row sum's reciprocal and the products
with it), the same in both maps; g by 2 u and the products g v are summed in 64 bits: 16 u of |g| . |v|.  r^3: three times 14 u of the outputs behind it and 3 u of
its square root and quotient.  eps and the result are rounded to fp32: 2 u.  16 + 51 + 2 = 69 u of r^3 eps |g| . |v|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _case(lens_q, lens_k, one, H, Hkv, hd, causal, ids=None, padded=False, tail=0, seed=0):
    """one: {query row: its key's row}, the rows that have a gradient."""
    from rectools_amd import ops

    g = torch.Generator().manual_seed(seed + hd)
    nq, nk, c, eps = sum(lens_q) + tail, sum(lens_k), 0.64, 1e-5
    q, k, v, gy = (torch.randn(n, h * 2 * hd, generator=g) for n, h in ((nq, H), (nk, Hkv), (nk, Hkv), (nq, H)))
    lam, w = torch.rand(H, generator=g) * 0.8 + 0.1, 1.0 + 0.1 * torch.randn(2 * hd, generator=g)
    rows, keys = torch.tensor(list(one.keys())), torch.tensor(list(one.values()))
    gy[[i for i in range(nq) if i not in one]] = 0.0
    G = gy[rows].view(-1, H, 2 * hd).double() * c * w.double()
    V = v[keys].view(-1, Hkv, 2 * hd).double()[:, torch.arange(H) // (H // Hkv)]
    r3 = (((1.0 - lam.double())[:, None] * V).square().mean(-1) + eps) ** -1.5 * eps
    want, size = -(r3 * (G * V).sum(-1)).sum(0), (r3 * (G * V).abs().sum(-1)).sum(0)
    cu = [None if padded else torch.tensor([0] + n).cumsum(0).cuda() for n in (lens_q, lens_k)]
    ts = [t.cuda().requires_grad_() for t in (q, k, v)]
    ld = lam.cuda().requires_grad_()
    y = ops.diff_attention(*ts, ld, *cu, len(lens_q), H, Hkv, max(lens_q), max(lens_k), causal, key_ids=None if ids is None else ids.cuda(), norm_w=w.cuda(), out_scale=c, eps=eps)
    got = torch.autograd.grad(y, ld, gy.cuda())[0].cpu().double()
    off = (got - want).abs()
    assert (off <= 69 * U * size).all(), (got, want, float((off / (69 * U * size)).max()))


@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 7), (2, 2, 32), (4, 2, 64), (8, 4, 20), (2, 1, 48)])
@pytest.mark.parametrize("causal", [True, False])
def test_sessions_of_one_row(H, Hkv, hd, causal):
    for B in (1, 2, 37, 200):
        _case([1] * B, [1] * B, {i: i for i in range(B)}, H, Hkv, hd, causal, padded=B == 37, seed=B)


@pytest.mark.parametrize("hd", [32, 50, 64])
def test_first_rows_of_sessions(hd):
    """Sessions without rows between them, rows behind the last one, a session in two halves of the keys."""
    lens = [0, 1, 5, 0, 0, 70, 1, 3, 0]
    _case(lens, lens, {0: 0, 1: 1, 6: 6, 76: 76, 77: 77}, 2, 1, hd, True, tail=0)
    lens = [600, 33]
    _case(lens, lens, {0: 0, 600: 600}, 2, 2, hd, True)
    _case([3, 1], [1, 1], {2: 0, 3: 1}, 2, 2, hd, True, tail=4)      # (more rows than keys: the first ones see none)
    _case([3, 1], [1, 1], {0: 0, 1: 0, 2: 0, 3: 1}, 2, 2, hd, False, tail=4)


@pytest.mark.parametrize("hd", [25, 32, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_one_key_left_by_the_mask(hd, causal):
    L, B = 200, 4
    ids = torch.zeros(B, L, dtype=torch.int64)
    ids[0, 199] = ids[1, 0] = ids[2, 90] = 5
    ids[3] = 1
    rows = {199: 199, 200: 200, 250: 200, 399: 200, 490: 490, 599: 490}
    _case([L] * B, [L] * B, rows, 2, 1, hd, causal, ids=ids.reshape(-1), padded=True)


@pytest.mark.parametrize("hd", [32, 64])
def test_one_key_of_split_keys(hd):
    ids = torch.zeros(3_000, dtype=torch.int64)
    ids[1_234] = 1
    _case([20], [3_000], {i: 1_234 for i in range(20)}, 2, 1, hd, True, ids=ids)
