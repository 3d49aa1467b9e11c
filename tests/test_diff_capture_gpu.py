"""A captured backward pass beside an eager graph of the same leaves is refused as well where the operator reads a leaf through a dense copy: the copy's
gradient goes on to the leaf's node, which belongs to the default stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cases():
    from rectools_amd import ops

    g = torch.Generator().manual_seed(2)
    wide = lambda: torch.randn(64, 8, generator=g).cuda().t()      # [8, 64], columns 8 elements apart      # noqa: E731
    pos, freq = torch.arange(8, device="cuda"), ops.rotary_frequencies(16, device="cuda")[0]
    lam, x = torch.full((2,), 0.3, device="cuda"), torch.randn(8, 64, generator=g).cuda()
    return {
        "rotary": (wide(), lambda t: ops.rotary(t, pos, freq, 4)),
        "keys": (wide(), lambda t: ops.rotary_qk(x, t, pos, freq, 4, 4)[1]),
        "lambda": (torch.randn(16, 2, generator=g).cuda().t(), lambda t: ops.diff_lambda(t, t, t, t, 0.3)),
        "attention": (wide(), lambda t: ops.diff_attention(t, x, x, lam, None, None, 1, 2, 2, 8, 8, True)),
        "norms": (wide(), lambda t: ops.norm_gate_residual(x, x, gate=t)[0]),
    }


@pytest.mark.parametrize("name", ["rotary", "keys", "lambda", "attention", "norms"])
def test_refused_beside_an_eager_graph_and_captured_without_it(name):
    leaf, call = _cases()[name]
    leaf = leaf.requires_grad_()
    assert leaf.is_leaf and not leaf.is_contiguous()

    def step():
        y = call(leaf)
        return torch.autograd.grad(y, leaf, torch.ones_like(y))[0]

    want = step()
    alive = call(leaf)
    with pytest.raises(RuntimeError, match="same leaf tensors"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    assert torch.equal(torch.autograd.grad(alive, leaf, torch.ones_like(alive))[0], want)
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(step(), want)
