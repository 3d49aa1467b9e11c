"""Sizes that the differential stack's C entries cannot count (heads and columns are 32-bit there): refused, not cut off.  Tensors without rows, so nothing is
allocated; with rows they would be answered for the columns that are left of the count."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [2 ** 31, 2 ** 32 + 64])
def test_columns_beyond_32_bits(cols):
    from rectools_amd import ops

    x, pos = torch.empty(0, cols, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    freq = ops.rotary_frequencies(16, device="cuda")[0]
    small = torch.empty(0, 64, device="cuda")
    for call in (lambda: ops.rotary(x, pos, freq, 1), lambda: ops.rotary(x, pos, freq, cols // 64), lambda: ops.rotary_qk(small, x, pos, freq, 1, cols // 64),
                 lambda: ops.diff_lambda(x, x, x, x, 0.1), lambda: ops.diff_lambda(*[torch.empty(1, 1, device="cuda").expand(cols, 1)] * 4, 0.1)):
        with pytest.raises((NotImplementedError, ValueError)):
            call()
    with pytest.raises(ValueError):      # (a product of heads and columns that wraps)
        ops.rotary_qk(small, small, pos, freq, 1, 2 ** 57)
    assert ops.rotary_qk(small, torch.empty(0, 128, device="cuda"), pos, freq, 1, 2)[1].shape == (0, 128)
