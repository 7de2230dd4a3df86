"""Calls around routed experts that are refused, each for its own reason, without a GPU."""
import os

import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_sinkhorn_b200 import _lib


@pytest.fixture(scope="module")
def ex():
    if not os.path.exists(_lib.library_path()):
        import __graft_entry__
        __graft_entry__.build()
    from flash_sinkhorn_b200 import experts
    return experts


def held(ex, e, n, k):
    return ex.Blocks8(torch.zeros(e, n, k, dtype=torch.float8_e4m3fn), torch.ones(e, -(-n // 128), -(-k // 128)))


def test_a_tangent_of_scales_is_refused(ex):
    """Products have no rule for it, and it would be dropped without a word."""
    q, x, off = held(ex, 2, 8, 16), torch.zeros(6, 16, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(q.scales, torch.ones_like(q.scales))
        with pytest.raises(ValueError, match="scales must not have a forward-mode tangent"):
            ex.grouped_mm8(x, ex.Blocks8(q.codes, dual), off)
