"""The attention operators at the edges of what their calls allow, against their definitions in 64 bits."""
import math

import pytest
import torch
from test_attention_gpu import DEV, make_cache

from swann_b200 import attention as A

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_a_pool_without_pages_beside_lengths_on_any_boundary():
    """Copies of nothing take an address from the lengths, which lie on 4-byte boundaries only."""
    k = torch.empty((0, 2, 16, 64), dtype=torch.float16, device=DEV)
    q = torch.randn((700, 4, 64), device=DEV).half()
    for B, slots in ((1, 3), (700, 3), (1, 4000)):       # by runs, a warp a pair, runs of several units
        table = torch.zeros((B, slots // 16 + 1), dtype=torch.int32, device=DEV)
        for at in (1, 2, 3):
            L = torch.full((B + 4,), slots, dtype=torch.int32, device=DEV)[at:at + B]
            parts = [A.decode(q[:B], k, k, table, L), A.decode(q[:B, :2], k, k, table, L)]
            if B == 1:
                parts.append(A.prefill(q[:3], k, k, table, ints(0, 3), L))
            for out, lse in parts:
                assert (out == 0).all() and (lse == -math.inf).all()
