"""How near differential attention comes to 64 bits, per tensor in the 2-norm: every route of the kernels (whole sessions, two halves of the keys, split
keys, few queries, shares of the keys) at the tolerance of test_diff_zero_rows_gpu.py, a few 1e-6 of a tensor's size.  A bound per element has to allow
for the worst case of every sum, 1e-4 and more; a lost half of an operand (1e-4), a wrong unit or a logarithm rounded at its size passes there.  What the
tolerance sees is tested on the CPU, with the mistake in the formulas."""
import math

import pytest
import torch

from test_diff_zero_rows_gpu import U, _check, _inputs, _plain


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,norm", [(2, 2, 32, True), (4, 2, 64, False), (1, 1, 25, True), (3, 1, 48, True), (2, 1, 9, False)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[200], [1, 2, 31, 32, 33], [90, 64, 129, 7]])
def test_whole_sessions(lens, causal, H, Hkv, hd, norm):
    n = sum(lens)
    ins, gy, _ = _inputs(n, n, H, Hkv, hd, norm, seed=n)
    _check(ins, gy, lens, lens, H, Hkv, causal)
    _check(ins, None, lens, lens, H, Hkv, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("size", [1.0, 1e-4])
def test_long_sessions_small_gradients(hd, size):
    lens = [600, 289]
    ins, gy, _ = _inputs(889, 889, 2, 1, hd, True, seed=4)
    _check(ins, gy * size, lens, lens, 2, 1, True)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 50, 64])
@pytest.mark.parametrize("rows", [[1], [3, 1], [12, 5], [20], [40, 2]])
def test_few_queries(rows, hd):
    """One session length: splits; lengths of a long tail: shares."""
    for keys in ([3_000] * len(rows), [4_000, 70][:len(rows)]):
        ins, _, _ = _inputs(sum(rows), sum(keys), 2, 1, hd, True, seed=sum(rows))
        _check(ins, None, rows, keys, 2, 1, True)
        _check(ins, None, rows, keys, 2, 1, False)


@pytest.mark.gpu
def test_split_keys_training():
    ins, gy, _ = _inputs(20, 2_000, 2, 1, 32, True, seed=9)
    _check(ins, gy, [20], [2_000], 2, 1, True)


@pytest.mark.gpu
@pytest.mark.parametrize("sharp", [0.05, 4.0])
def test_flat_and_sharp_maps(sharp):
    lens = [65, 130]
    ins, gy, _ = _inputs(195, 195, 2, 2, 32, True, seed=6)
    ins[0] = ins[0] * sharp
    _check(ins, gy, lens, lens, 2, 2, True)


def _one_half(t):
    """The leading half of a split operand: 11 bits."""
    m, e = torch.frexp(t)
    return torch.ldexp((m * 2048.0).round() / 2048.0, e)


@pytest.mark.parametrize("which,seen_by", [(0, "y"), (0, "dk"), (1, "y"), (1, "dq"), (2, "y"), (2, "dq"), (5, "dv"), (5, "dk"), (5, "dlam")])
def test_the_tolerance_sees_a_lost_half(which, seen_by):
    """which: q, k, v, or 5: dy."""
    lens = [90, 33]
    ins, gy, _ = _inputs(123, 123, 2, 1, 32, True, seed=8)
    args = (lens, lens, 2, 1, True, 0.64, 1e-5)
    want, near = (_plain(ins, gy, *args, t) for t in (torch.float64, torch.float32))
    g = torch.Generator().manual_seed(1)
    moved = [_plain(ins, gy, *args, torch.float64, g) for _ in range(4)]
    lost = [None if t is None else _one_half(t) if i == which else t for i, t in enumerate(ins)]
    bad = _plain(lost, _one_half(gy) if which == 5 else gy, *args, torch.float64)
    for n in want:
        rms = math.sqrt(sum(float((m[n] - want[n]).square().sum()) for m in moved) / 4)
        allowed = 3 * rms + 3 * float((near[n].double() - want[n]).norm()) + 16 * U * float(want[n].norm())
        assert n == "dlam" or allowed < 1e-5 * float(want[n].norm())      # (dlam: one number per head, what is left of its rows' shares)
        if n == seen_by:
            assert float((bad[n] - want[n]).norm()) > 5 * allowed
