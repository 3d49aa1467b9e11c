"""Where a differential layer stack starts: the vectors behind lam keep their deviation of 0.1 through the models' initialisation, which draws every matrix anew."""
import math

import pytest
import torch

from rectools_amd import lightning as hl
from rectools_amd import nn as hnn


def _starts(layers):
    """The vectors' deviation and lam of every head against its block's lambda_init."""
    blocks = list(layers.transformer_blocks)
    vectors = torch.cat([getattr(b, n).detach().cpu().double().reshape(-1) for b in blocks for n in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2")])
    # n samples: the deviation is off by 0.1 / sqrt(2 n), 5 of these
    assert abs(float(vectors.std()) - 0.1) < 5 * 0.1 / math.sqrt(2 * vectors.numel()) and abs(float(vectors.mean())) < 5 * 0.1 / math.sqrt(vectors.numel())
    for b in blocks:
        q1, k1, q2, k2 = (getattr(b, n).detach().cpu().double() for n in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"))
        lam = torch.exp((q1 * k1).sum(1)) - torch.exp((q2 * k2).sum(1)) + b.lambda_init
        # a product of two vectors has a deviation of 0.01 sqrt(hd); lam the difference of two: 5 of these (exp(x) - 1 < 1.4 x up to there)
        assert (lam - b.lambda_init).abs().max() < 1.4 * 5 * math.sqrt(2) * 0.01 * math.sqrt(b.hd)
    return blocks


@pytest.mark.parametrize("H,kv", [(4, 4), (8, 2), (2, 1)])
def test_lambda_vectors_keep_their_deviation(H, kv):
    torch.manual_seed(3)
    layers = hnn.DifferentialTransformerLayers(3, 256, H, 0.1, n_kv_heads=kv)
    before = {n: t.detach().clone() for n, t in layers.named_parameters()}
    hl.xavier_normal_init(layers)
    for n, t in layers.named_parameters():
        assert torch.equal(t, before[n]) == ("lambda" in n or t.dim() < 2), n
    _starts(layers)


def test_other_stacks_draw_as_before():
    """Matrices in the order of the parameters, nothing between them."""
    torch.manual_seed(3)
    layers = hnn.PreLNTransformerLayers(2, 64, 2, 0.1)
    torch.manual_seed(5)
    hl.xavier_normal_init(layers)
    torch.manual_seed(5)
    for n, t in layers.named_parameters():
        if t.dim() > 1:
            assert torch.equal(t, torch.nn.init.xavier_normal_(torch.empty_like(t))), n


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["sasrec", "bert"])
def test_a_fitted_model_started_there(family):
    """lr so small that the vectors are where fit() put them."""
    from rectools_amd import models as M
    from test_diff_layers_gpu import _dataset

    cls = M.SASRecModel if family == "sasrec" else M.BERT4RecModel
    m = cls(n_factors=256, n_blocks=2, n_heads=4, session_max_len=24, lr=1e-12, batch_size=48, dropout_rate=0.1, loss="softmax", epochs=1, seed=1, deterministic=True,
            use_key_padding_mask=True, transformer_layers_type=hnn.DifferentialTransformerLayers).fit(_dataset())
    _starts(m.torch_model.transformer_layers)


@pytest.mark.parametrize("H,kv,d", [(4, 0, 64), (4, -1, 64), (4, -4, 64), (0, None, 64), (-2, -1, 64), (4, 2, 0), (2, 1, -64)])
def test_counts_that_are_not_positive_are_refused(H, kv, d):
    with pytest.raises(ValueError):
        hnn.DifferentialTransformerLayers(1, d, H, 0.0, n_kv_heads=kv)
