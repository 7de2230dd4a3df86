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


@pytest.mark.parametrize("n,k", [(1, 1), (1, 5), (2, 2), (2, 3), (3, 3), (4, 4), (2, 64), (5, 2)])
def test_few_rows(ortho, n, k):
    """Nothing averages: one singular value is off by at most 2e-2 (test_gpu_orthogonalize.py), and roundings of several entries, each at most u of
    its own, are an error matrix whose 2-norm is up to sqrt(rows) times that of one, of which two rows can come together: 2e-2 sqrt(2), with the
    result's own rounding of 2^-11 less than the 3 % that are documented."""
    m = normal(gen(n + 10 * k), 100_000, n, k)
    assert relative(ortho(m, dtype=FP16), plain(m)) <= 3e-2


@pytest.mark.parametrize("n,k", [(64, 64), (200, 300), (512, 256), (700, 1024)])
def test_where_singular_values_go(ortho, n, k):
    """From 0.003 on to between 0.6818 and 1.2024 in exact arithmetic (extremes of the steps' polynomial there); 0.5 % for roundings."""
    g, r = gen(n), min(n, k)
    u, v = torch.linalg.qr(normal(g, n, r))[0], torch.linalg.qr(normal(g, k, r))[0]
    spread = max(a for a in (0.5, 1.0, 1.5, 2.0) if 10**-a / torch.logspace(-a, 0, r).norm() >= 0.0031)
    m = (u * torch.logspace(-spread, 0, r, device="cuda")) @ v.T
    values = torch.linalg.svdvals(ortho(m, dtype=FP16).double())[:r]
    assert values.max() <= 1.2024 * 1.005 and values.min() >= 0.6818 * 0.995


@pytest.mark.parametrize("batch,n,k", [(3, 140, 90), (3, 1, 50), (3, 600, 600), (40, 130, 1000), (30, 700, 512)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_matrix_with_a_value_that_is_not_finite_gives_nan_throughout(ortho, batch, n, k, value):
    m = normal(gen(n), batch, n, k)
    want = ortho(m)
    m[1, n // 2, k - 1] = value
    for steps in (1, 5):
        y = ortho(m, steps=steps)
        assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()
    assert torch.equal(y[[0, 2]], want[[0, 2]])
