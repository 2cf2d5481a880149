"""Values that would give wrong numbers without a word are refused (CPU)."""

from __future__ import annotations

import pytest
import torch

from flash_head.sampling import sample_logits
from flash_head.w4 import W4Weight
from test_sampling_host import fake


@pytest.mark.parametrize("k", [2.5, 0.5])
def test_a_top_k_between_integers(k):
    x, u = fake(torch.zeros(2, 8)), torch.zeros(2, dtype=torch.float64)
    with pytest.raises(ValueError, match="integer"):
        sample_logits(x, u, top_k=k)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_weight_that_is_not_finite(bad, zeros):
    """Its group's scale would be infinite, and 0 times that no number."""
    w = torch.ones(6, 128, dtype=torch.bfloat16)
    w[4, 70] = bad
    with pytest.raises(ValueError, match="finite"):
        W4Weight.from_dense(w, 64, zeros)


@pytest.mark.parametrize("dtype,big", [(torch.float16, 4096.0), (torch.bfloat16, 2.0 ** 124)])
def test_row_factors(dtype, big):
    """Rows whose weights may pass the type's largest number are brought down by
    2^-4, all others are not touched, whatever their scales are."""
    s = torch.tensor([[0.01], [big], [big * 1.5], [torch.finfo(dtype).max], [2.0 ** -24],
                      [0.0], [float("inf")], [float("nan")]]).to(dtype)
    w = W4Weight.from_quantized(torch.zeros(8, 16, dtype=torch.uint8), s)
    assert w.row_mul[:8].tolist() == [1, 1, 2.0 ** -4, 2.0 ** -4, 1, 1, 1, 1]
    assert (w.row_mul[8:] == 1).all() and w.row_mul.shape == (128,)
    top = (s.float() * w.row_mul[:8].view(8, 1)).to(dtype).float()
    fine = torch.isfinite(s.float())
    assert torch.isfinite((top * 15).to(dtype).float())[fine].all()
