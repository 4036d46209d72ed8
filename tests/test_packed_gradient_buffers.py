"""Buffers for the gradients of packed attention: all three or none."""
import itertools

import pytest
import torch

from flame_amd import capi


@pytest.mark.parametrize("given", [g for g in itertools.product([False, True], repeat=3) if 0 < sum(g) < 3])
def test_some_buffers(given):
    """Of fewer than three none would be written, and nothing would say so."""
    q, k = torch.zeros((10, 4, 64), dtype=torch.bfloat16), torch.zeros((10, 2, 64), dtype=torch.bfloat16)
    cu, lse = torch.tensor([0, 10], dtype=torch.int32), torch.zeros((4, 10))
    grads = tuple(t.clone() if g else None for t, g in zip((q, k, k), given))
    with pytest.raises(AssertionError, match="all three gradients or none"):
        capi.attn_packed_bwd(q, k, k, q, q, lse, cu, cu, 0.1, grads=grads)
