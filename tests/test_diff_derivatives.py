"""Derivatives that the differential stack's operators have not got are refused, never dropped in silence."""
import pytest
import torch
from torch.autograd import forward_ad

from rectools_amd import ops


def _calls(dev):
    """[(name, tensors, call)]: every tensor that a result depends on smoothly."""
    g = torch.Generator().manual_seed(1)
    new = lambda *shape: torch.randn(*shape, generator=g).to(dev)      # noqa: E731
    x, w = new(6, 64), new(64)
    freq, pos = ops.rotary_frequencies(16, device=dev)[0], torch.arange(6, device=dev)
    return [
        ("rotary", [x], lambda q: ops.rotary(q, pos, freq, 4)),
        ("rotary_qk", [x, new(6, 32)], lambda q, k: ops.rotary_qk(q, k, pos, freq, 4, 2)),
        ("rotary frequencies", [freq], lambda f: ops.rotary(x, pos, f, 4)),
        ("diff_lambda", [new(2, 16) for _ in range(4)], lambda *t: ops.diff_lambda(*t, 0.3)),
        ("diff_attention", [x, x, x, new(2), new(32)], lambda q, k, v, lam, n: ops.diff_attention(q, k, v, lam, None, None, 1, 2, 2, 6, 6, True, norm_w=n)),
        ("norm_gate_residual", [x, x, x, w, w, w, w, w],
         lambda x, f, z, s, pw, pb, nw, nb: ops.norm_gate_residual(x, f, gate=z, post=(pw, pb), scale=s, pre=(nw, nb), kind="layer")),
    ]


def _refused(dev):
    for name, tensors, call in _calls(dev):
        for i, t in enumerate(tensors):
            for grad in (False, True):
                with forward_ad.dual_level():
                    args = [u.detach().clone() for u in tensors]
                    args[i] = forward_ad.make_dual(args[i].requires_grad_(grad), torch.ones_like(t))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*args)
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*args)


def test_forward_mode_is_refused():
    _refused("cpu")


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_device():
    _refused("cuda")
    for _, tensors, call in _calls("cuda"):
        call(*tensors)      # (and nothing else is)
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(lambda *t: call(*t), tuple(tensors), tuple(torch.ones_like(t) for t in tensors))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_frequencies_that_require_a_gradient_are_refused(dev):
    x, pos = torch.randn(6, 64, device=dev), torch.arange(6, device=dev)
    freq = ops.rotary_frequencies(16, device=dev)[0].requires_grad_()
    for call in (lambda: ops.rotary(x, pos, freq, 4), lambda: ops.rotary_qk(x, x, pos, freq, 4, 4)):
        with pytest.raises(NotImplementedError, match="frequencies"):
            call()
    if dev == "cuda":
        with torch.no_grad():
            assert torch.equal(ops.rotary(x, pos, freq, 4), ops.rotary(x, pos, freq.detach(), 4))
