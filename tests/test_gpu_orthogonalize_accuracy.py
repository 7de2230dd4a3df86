"""What the lower part of X keeps in an orthogonal update, and where singular values go."""
import pytest
import torch

from test_gpu_experts import FP16, gen, normal
from test_gpu_orthogonalize import plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ortho():
    from flash_sinkhorn_b200.experts import orthogonalize
    return orthogonalize


def relative(got, want):
    return ((got.double() - want).square().sum((-2, -1)) / want.square().sum((-2, -1))).sqrt().max().item()


@pytest.mark.parametrize("n,k", [(300, 700), (512, 512), (900, 260), (2048, 1024)])
def test_roundings_along_small_singular_values(ortho, n, k):
    """Of a matrix of rank one nearly all of a rounding lies along singular values of 0, which a step multiplies by 3.4445.

    An fp16 value is off by 2^-10 / sqrt(12) / m in the mean square, m in [1, 2) its mantissa: 2^-10 * 0.289 * 0.736 = 2.07e-4 of it. The
    singular value goes 1, 0.70, 1.11, 0.72, 1.09, 0.73, so with X rounded to one fp16 value before the last step the result is
    off by 3.4445 * 2.07e-4 * 1.09 / 0.73 = 1.06e-3 of its norm, and by 2.07e-4 for its own rounding: 1.08e-3. Roundings of A and of P along one direction
    average over n entries (1e-4). Half of that more is allowed; a rounding before the last step but one leaves 2.4e-3.
    """
    g = gen(n)
    m = normal(g, 2, n, 1) @ normal(g, 2, 1, k)
    assert relative(ortho(m, dtype=FP16), plain(m)) <= 1.6e-3


@pytest.mark.parametrize("n,k", [(128, 1000), (129, 1000), (1000, 128), (90, 2048)])
def test_stacks_of_few_rows(ortho, n, k):
    """Stacks too large for one launch, matrices whose rows fill one CTA of a pair or not even that; the bound is that of all updates."""
    from test_gpu_orthogonalize import check
    m = normal(gen(n + k), 40, n, k)
    check(ortho(m), plain(m))
