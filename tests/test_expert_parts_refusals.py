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


@pytest.mark.parametrize("w_in,w_out", [((2, 96, 64), (2, 72, 48)), ((2, 96, 64), (2, 56, 48)), ((2, 96, 64), (3, 64, 48)), ((2, 96, 64), (2, 64, 40)),
                                        ((2, 96, 72), (2, 64, 48)), ((2, 95, 64), (2, 64, 47))])
def test_held_weights_of_a_layer_fit_one_another(ex, w_in, w_out):
    """Also where the sums back into tokens would come out with another width than the rows."""
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    r = ex.Routing(torch.zeros(3, 2), *[torch.zeros(3, 2, dtype=torch.int32)] * 5)
    with pytest.raises(ValueError, match=r"w_in \[E, 2 F, D\] and w_out \[E, D, F\]"):
        ex.expert_mlp(x, held(ex, *w_in), held(ex, *w_out), r)
