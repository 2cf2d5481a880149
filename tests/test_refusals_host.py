"""Values that would give wrong numbers without a word are refused (CPU)."""

from __future__ import annotations

import pytest
import torch

from flash_head.sampling import sample_logits
from test_sampling_host import fake


@pytest.mark.parametrize("k", [2.5, 0.5])
def test_a_top_k_between_integers(k):
    x, u = fake(torch.zeros(2, 8)), torch.zeros(2, dtype=torch.float64)
    with pytest.raises(ValueError, match="integer"):
        sample_logits(x, u, top_k=k)
