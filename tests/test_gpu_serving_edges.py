"""Edges of the shared-prefix attention, the scored attention and the budgeted cache on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def test_scores_where_keys_times_heads_pass_32_bits(lsa):
    """64 heads on a cache of just over 2^25 keys: all logits are zero, so every key - the first ones
    among them - gains 64 / n. The weight is a sum of 64 fp32 terms of relative error below 2e-4."""
    n = (1 << 25) + 300
    k = torch.zeros(1, n, 1, 64, dtype=BF, device=DEV)
    q = torch.ones(1, 1, 64, 64, dtype=BF, device=DEV)
    scores = torch.zeros(1, 1, n, device=DEV)
    out, got = lsa.scored_attention(q, k, k, torch.tensor([n], device=DEV), scores)
    assert (out == 0).all()
    assert float((got.double() * n / 64 - 1).abs().max()) <= 2e-4
