"""Host side of the differential-attention stack's operators, without a GPU: frequencies, workspace arithmetic, refusals of the C entries (no
launch is reached) and of the layer stack."""
import math

import pytest
import torch

from rectools_amd import _lib, ops

INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 4
P = 1 << 20      # a non-null address that is never read


def test_frequencies():
    f, gain = ops.rotary_frequencies(8)
    assert f.dtype == torch.float64 and gain == 1.0
    torch.testing.assert_close(f, torch.tensor([10_000.0 ** (-2 * j / 8) for j in range(4)], dtype=torch.float64), rtol=1e-15, atol=0)
    g, _ = ops.rotary_frequencies(8, scaling="linear", factor=4.0)
    torch.testing.assert_close(g, f / 4, rtol=1e-15, atol=0)
    b, _ = ops.rotary_frequencies(8, scaling="base", factor=4.0)
    assert float(b[0]) == 1.0 and abs(float(b[-1] * 4 / f[-1]) - 1) < 1e-12      # the fastest pair stays, the slowest is stretched by the factor
    p, gain = ops.rotary_frequencies(64, scaling="parts", factor=4.0, trained_len=4096)
    q, _ = ops.rotary_frequencies(64)
    turns = 4096 * q / (2 * math.pi)
    assert torch.equal(p[turns >= 32], q[turns >= 32]) and torch.equal(p[turns <= 1], q[turns <= 1] / 4) and abs(gain - (0.1 * math.log(4) + 1)) < 1e-15
    assert ((p <= q) & (p >= q / 4)).all()
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, scaling="x"), dict(rot=8, factor=0.5), dict(rot=8, base=1.0), dict(rot=8, trained_len=0), dict(rot=8, factor=float("nan"))):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


def test_rotary_refuses():
    def call(n=2, kv=2, M=4, hd=16, rot=8, q=P, ld=32, pos=P, freq=P):
        return _lib.load().rt_rotary(q, ld, q, ld, n, P, 32, P, 32, kv, pos, freq, M, hd, rot, 0, 1.0, 0, None)

    for kw in (dict(rot=7), dict(rot=18), dict(rot=0), dict(hd=0), dict(M=-1), dict(n=-1), dict(q=None), dict(ld=31), dict(pos=None), dict(freq=None)):
        assert call(**kw) == INVALID, kw
    assert call(M=0) == 0 and call(n=0, kv=0) == 0


def _fwd(B=2, H=2, Hkv=2, hd=16, Lq=4, Lk=4, Nq=8, Nk=8, cu_q=None, cu_k=None, q=P, k=P, lam=P, y=P, ld=64, ldk=64, saved=None, sn=0, ws=None, n=0):
    return _lib.load().rt_diffattn_fwd(q, ld, k, ldk, P, ldk, lam, cu_q, cu_k, None, B, H, Hkv, hd, Lq, Lk, Nq, Nk, 0.0, 1, None, 1.0, 1e-5, y, ld, saved, sn, ws, n, None)


def test_attention_refuses():
    for kw in (dict(H=3), dict(H=0), dict(Hkv=0), dict(hd=0), dict(B=-1), dict(Nq=7), dict(Nk=9), dict(q=None), dict(k=None), dict(lam=None), dict(y=None),
               dict(ld=63), dict(ldk=63), dict(Lq=-1), dict(Nq=-8)):
        assert _fwd(**kw) == INVALID, kw
    assert _fwd(hd=65, ld=260, ldk=260) == UNSUPPORTED
    assert _fwd(B=0, Nq=0, Nk=0) == 0
    lib = _lib.load()
    saved = lib.rt_diffattn_saved_bytes(2, 2, 16, 8, 8)
    assert saved > 0 and lib.rt_diffattn_saved_bytes(2, 2, 65, 8, 8) == 0
    for kw in (dict(saved=P, sn=saved - 1), dict(saved=P + 4, sn=saved)):
        assert _fwd(**kw) == WORKSPACE, kw
    need = lib.rt_diffattn_fwd_workspace_bytes(1, 2, 2, 16, 1, 100_000, 1, 100_000, 0)
    assert 0 < need < 100_000 * 64 and lib.rt_diffattn_fwd_workspace_bytes(64, 2, 2, 16, 200, 200, 12_800, 12_800, 1) == 0      # (one query: no planes)
    assert lib.rt_diffattn_fwd_workspace_bytes(64, 2, 2, 16, 200, 200, 12_800, 12_800, 0) > 12_800 * 2 * 3 * 128
    big = dict(B=1, Lq=1, Lk=100_000, Nq=1, Nk=100_000)
    assert _fwd(**big) == WORKSPACE and _fwd(**big, ws=P, n=need - 1) == WORKSPACE
    assert lib.rt_diffattn_fwd_workspace_bytes(0, 2, 2, 16, 1, 1, 1, 1, 0) == 0 and lib.rt_diffattn_fwd_workspace_bytes(1, 3, 2, 16, 1, 1, 1, 1, 0) == 0

    def bwd(sv=P, sn=1 << 30, ws=P, n=1 << 30, Nq=8, norm_w=None, dw=None, dlam=P, dy=P, dq=P, dk=P):
        return lib.rt_diffattn_bwd(sv, sn, P, None, None, None, 2, 2, 2, 16, 4, 4, Nq, 8, 0.0, 1, norm_w, 1.0, 1e-5, dy, 64, dq, 64, dk, 64, P, 64, dlam, dw, ws, n, None)

    for kw in (dict(ws=None), dict(ws=P + 8), dict(n=lib.rt_diffattn_bwd_workspace_bytes(2, 16, 8) - 1), dict(sv=None), dict(sn=saved - 1), dict(sv=P + 4)):
        assert bwd(**kw) == WORKSPACE, kw
    for kw in (dict(Nq=7), dict(norm_w=P), dict(dw=P), dict(dlam=None), dict(dy=None), dict(dq=None), dict(dk=None)):
        assert bwd(**kw) == INVALID, kw


def test_lambda_refuses():
    lib = _lib.load()
    assert lib.rt_diff_lambda_fwd(None, P, P, P, 0.1, 2, 4, P, None) == INVALID and lib.rt_diff_lambda_fwd(P, P, P, P, 0.1, 2, 0, P, None) == INVALID
    assert lib.rt_diff_lambda_fwd(None, None, None, None, 0.1, 0, 4, None, None) == 0
    assert lib.rt_diff_lambda_bwd(P, P, P, P, P, 2, 4, P, P, P, None, None) == INVALID


def test_norm_gate_refuses():
    lib = _lib.load()

    def fwd(x=P, f=P, y=P, h=None, pw=None, pb=None, nw=None, nb=None, M=4, d=8, p=0.0, stat=None):
        return lib.rt_norm_gate_fwd(x, f, None, None, pw, pb, nw, nb, 0, 1.0, 1e-5, p, 0, 0, M, d, y, h, stat, None)

    for kw in (dict(x=None), dict(f=None), dict(y=None), dict(h=P), dict(nw=P), dict(pb=P), dict(nb=P), dict(M=-1), dict(d=0), dict(p=1.0), dict(p=-0.5), dict(p=float("nan")),
               dict(stat=P + 4)):
        assert fwd(**kw) == INVALID, kw
    assert fwd(d=8193) == UNSUPPORTED and fwd(M=0, x=None) == 0

    def bwd(f=P, stat=P, dx=P, dz=None, gh=None, ws=P, n=1 << 30):
        return lib.rt_norm_gate_bwd(P, gh, None, f, None, None, None, None, None, 0, 1.0, 0.0, 0, 0, 4, 8, stat, dx, P, dz, P, None, None, None, None, ws, n, None)

    for kw in (dict(f=None), dict(stat=None), dict(dx=None), dict(dz=P), dict(gh=P)):
        assert bwd(**kw) == INVALID, kw
    assert bwd(ws=None) == WORKSPACE and bwd(n=3) == WORKSPACE
    assert lib.rt_norm_gate_bwd_workspace_bytes(100, 64) > 0 and lib.rt_norm_gate_bwd_workspace_bytes(0, 64) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    for bad in (lambda: ops.norm_gate_residual(x, x), lambda: ops.diff_lambda(x, x, x, x, 0.1), lambda: ops.rotary(x, torch.arange(4), torch.zeros(4, dtype=torch.float64), 4),
                lambda: ops.diff_attention(x, x, x, torch.zeros(2), None, None, 1, 2, 2, 4, 4, True)):
        with pytest.raises(_lib.HipLibraryError):
            bad()


def test_stack_refuses_and_keeps_its_frequencies_in_64_bits():
    from rectools_amd.nn import DifferentialTransformerLayers as S

    for bad in (dict(n_factors=30, n_heads=4), dict(n_factors=64, n_heads=4, n_kv_heads=3), dict(n_factors=64, n_heads=2, rotary_part=0.0),
                dict(n_factors=64, n_heads=2, rotary_part=1.5), dict(n_factors=64, n_heads=16, rotary_part=0.5, rotary_scaling="parts", rotary_factor=0.1)):
        with pytest.raises(ValueError):
            S(n_blocks=1, dropout_rate=0.0, **bad)
    with pytest.raises(NotImplementedError):
        S(1, 512, 2, 0.0)
    s = S(2, 64, 2, 0.0).double().float()
    assert s.rotary.freq.dtype == torch.float64 and not any("freq" in n for n in s.state_dict())
    assert s.packed_ok(64, 50, True, True) and not s.packed_ok(64, 50, True, False)
    cu = torch.tensor([0, 3, 3, 5])
    assert S._packed_positions(cu, 7).tolist() == [0, 1, 2, 0, 1, 0, 1]      # pylint: disable=protected-access
