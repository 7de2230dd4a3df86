"""8-bit products of short groups where every CTA takes several tiles: rows' factors pass from tile to tile."""
import pytest
import torch

from test_gpu_experts import BF16, gen, normal
from test_gpu_mm8 import blocks8, close, grouped, offsets_of, rows8, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    from flash_sinkhorn_b200 import experts
    return experts


@pytest.mark.parametrize("k", [64, 128, 300, 384, 640, 200])  # one, one, three, three, five and two blocks of 128
def test_many_tiles_of_odd_numbers_of_blocks(ex, k):
    """512 tiles and more for two CTAs an SM, groups of 17 to 32 rows whose scales differ from row to row by powers of two up to 2^12."""
    g = gen(k)
    e, n = 64, 1000
    counts = torch.randint(17, 33, (e,), generator=g, device="cuda").tolist()
    x = normal(g, sum(counts), k) * torch.exp2(torch.randint(-6, 7, (sum(counts), 1), generator=g, device="cuda").float())
    x, w, off = x.to(BF16), normal(g, e, n, k, scale=k**-0.5, dtype=BF16), offsets_of(counts)
    codes, scales = blocks8(w)
    want, size = grouped(rows8(x), codes * wide(scales, n, k), off[1:].tolist())
    q = ex.to_blocks8(w)
    first = ex.grouped_mm8(x, q, off)
    close(first, want, size, BF16)
    for _ in range(20):
        assert torch.equal(ex.grouped_mm8(x, q, off), first)


@pytest.mark.parametrize("mean", [17, 143, 145])
def test_gradient_to_rows_on_both_sides_of_its_choice(ex, mean):
    """Enough tiles of 256 x 256 for all CTAs, groups below and above the rows from which pairs take them."""
    g = gen(mean)
    e, n, k = 40, 264, 1100
    counts = [mean - 9, mean + 9] * (e // 2)
    x, off = normal(g, sum(counts), k, dtype=BF16).requires_grad_(), offsets_of(counts)
    w, dy = normal(g, e, n, k, scale=k**-0.5, dtype=BF16), normal(g, sum(counts), n, dtype=BF16)
    codes, scales = blocks8(w)
    (dx,) = torch.autograd.grad(ex.grouped_mm8(x, w, off), x, dy)
    close(dx, *grouped(rows8(dy), codes * wide(scales, n, k), off[1:].tolist(), transposed=True), BF16)
