"""Orthogonal updates against the definition in 64 bits.

Bound on the error, relative to the norm of the result. fp16 rounds by half a unit at most, u = 2^-11. In a step the roundings of A, of P and of
X's upper part enter a singular value s with (|b s^2 + 2 c s^4| + 2 |b s^2 + c s^4|) u s, 6.2 u at s = 1, and an error from before is
multiplied by a + 3 b s^2 + 5 c s^4.

One singular value (a matrix of one row or column): s goes 1, 0.70, 1.11, 0.72, 1.09, 0.73; new errors are at most 3.0e-3, 1.7e-3, 3.2e-3, 1.9e-3,
3.0e-3, factors 1.14, 1.30, 1.25, 0.80 in magnitude: 3.0e-3, 5.2e-3, 9.9e-3, 1.42e-2, 1.44e-2 of 0.73, or 2e-2.

More of them: roundings of many entries add as independent ones do, so each of the three counts with u / sqrt(3) in the mean and their squares add:
sqrt(0.7^2 + 2 * 2.74^2) u / sqrt(3) = 1.1e-3 for a step, and with the factors above 1.1e-3, 1.7e-3, 2.5e-3, 3.3e-3, 2.9e-3 of 0.73, or 4e-3, with 2.5 times
that allowed, since few entries average little and singular values take other ways: 1e-2. Half a unit for the rounding to the type besides.
"""
import pytest
import torch

from test_gpu_experts import BF16, FP16, FP32, ULP, gen, normal

pytestmark = pytest.mark.gpu
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def ortho():
    from flash_sinkhorn_b200.experts import orthogonalize
    return orthogonalize


def plain(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        m = x @ x.mT
        x = a * x + (b * m + c * m @ m) @ x
    return x.mT if tall else x


def check(got, want, dtype=BF16, off=None):
    assert got.dtype == dtype and got.shape == want.shape and got.is_contiguous()
    off = off or (2e-2 if 1 in got.shape[-2:] else 1e-2)
    diff = (got.double() - want).square().sum((-2, -1)).sqrt()
    norm = want.square().sum((-2, -1)).sqrt()
    assert (diff <= (off + ULP[dtype]) * norm).all(), (diff / norm).max().item()


SHAPES = [(1, 1, 1), (2, 1, 5), (1, 7, 1), (3, 16, 16), (1, 64, 65), (2, 65, 64), (1, 128, 128), (5, 129, 257), (2, 300, 501), (3, 501, 300), (1, 512, 512),
          (4, 640, 200), (40, 130, 100), (1, 260, 1000), (20, 256, 300), (12, 512, 700), (9, 700, 520)]


@pytest.mark.parametrize("batch,n,k", SHAPES)
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (FP32, BF16), (FP16, FP16)])
def test_orthogonalize(ortho, batch, n, k, dtype, out):
    g = normal(gen(n + k), batch, n, k, scale=1e-2, dtype=dtype)
    check(ortho(g, dtype=out), plain(g), out)


@pytest.mark.parametrize("n,k", [(96, 96), (512, 512), (300, 700)])
@pytest.mark.parametrize("kind", ["decaying", "low rank", "rank one", "one entry", "orthogonal"])
def test_uneven_singular_values(ortho, n, k, kind):
    """What small singular values come from keeps its bits: operands of 11 bits alone would leave errors of 1 to 10 %."""
    g = gen(n)
    if kind == "decaying":
        m = (normal(g, n, n // 4) * torch.logspace(0, -2, n // 4, device="cuda")) @ normal(g, n // 4, k) + 0.05 * normal(g, n, k)
    elif kind == "low rank":
        m = normal(g, n, n // 4) @ normal(g, n // 4, k)
    elif kind == "rank one":
        m = normal(g, n, 1) @ normal(g, 1, k)
    elif kind == "one entry":
        m = torch.zeros(n, k, device="cuda")
        m[n // 2, k // 3] = -3.0
    else:
        m = torch.linalg.qr(normal(g, k, n))[0].T
    check(ortho(m), plain(m))
    check(ortho(m.T), plain(m.T))


@pytest.mark.parametrize("steps", [1, 2, 8])
def test_steps_and_coefficients(ortho, steps):
    g = normal(gen(steps), 2, 200, 150)
    check(ortho(g, steps=steps), plain(g, steps), off=1.6e-2 if steps == 8 else None)  # three steps more
    cubic = (1.5, -0.5, 0.0)
    check(ortho(g, steps=steps, coefficients=cubic), plain(g, steps, cubic))


def test_magnitudes(ortho):
    """Sums of squares that 32 bits do not hold, and a norm next to eps."""
    g = normal(gen(3), 1, 70, 50)
    for scale in (1e30, 1e-15, 1e-7):
        check(ortho(g * scale), plain(g * scale))
    check(ortho(g * 1e-25, eps=1e-30), plain(g * 1e-25, eps=1e-30))


def test_zeros_and_values_that_are_not_finite_stay_in_their_matrix(ortho):
    g = normal(gen(4), 5, 140, 90)
    ref = ortho(g)
    g[1] = 0
    g[2, 7, 8], g[4, 139, 89] = float("inf"), float("nan")
    y = ortho(g)
    assert torch.equal(y[0], ref[0]) and torch.equal(y[3], ref[3])
    assert torch.equal(y[1], torch.zeros_like(y[1])) and torch.isnan(y[2]).any() and torch.isnan(y[4]).all()


def test_shapes_and_strides(ortho):
    g = gen(5)
    m = normal(g, 2, 3, 70, 90)
    y = ortho(m)
    check(y, plain(m))
    assert torch.equal(ortho(m[1, 2]), y[1, 2])
    assert torch.equal(ortho(m.mT.contiguous().mT), y)
    big = normal(g, 4, 80, 100)
    check(ortho(big[::2, 3:73, 5:95]), plain(big[::2, 3:73, 5:95]))
    check(ortho(m[0, :1].expand(3, 70, 90)), plain(m[0, :1].expand(3, 70, 90)))
    assert ortho(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    leaf = m.clone().requires_grad_()
    assert not ortho(leaf).requires_grad


def test_same_bits_on_another_stream_and_in_a_graph(ortho):
    m = normal(gen(6), 6, 300, 200, dtype=BF16)
    want = ortho(m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ortho(m)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, again)
    torch.cuda.synchronize()
    static, graph = m.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ortho(static)
    for seed in (1, 2):
        static.copy_(normal(gen(seed), 6, 300, 200, dtype=BF16))
        graph.replay()
        assert torch.equal(out, ortho(static))


@pytest.mark.parametrize("batch,n,k", [(1, 100, 150), (20, 512, 600)])
def test_updates_that_give_up(ortho, batch, n, k):
    """With no clocks to wait the result is NaN and the health word says so; afterwards all is as before."""
    from flash_sinkhorn_b200 import _lib
    lib = _lib.load()
    m = normal(gen(7), batch, n, k)
    want = ortho(m)
    assert lib.fs_device_error() == 0
    before = lib.fs_set_product_limit(0)
    try:
        y = ortho(m)
    finally:
        lib.fs_set_product_limit(before)
    assert torch.isnan(y).all() and lib.fs_device_error() == 1
    assert lib.fs_clear_device_error() == 0 and lib.fs_device_error() == 0
    assert torch.equal(ortho(m), want)


def test_refusals(ortho):
    m = torch.zeros(4, 5, device="cuda")
    for call in (lambda: ortho(m[0]), lambda: ortho(m.double()), lambda: ortho(m.cpu()), lambda: ortho(m, dtype=FP32), lambda: ortho(m, steps=0),
                 lambda: ortho(m, steps=65), lambda: ortho(m, coefficients=(1.0, 40.0, 0.0)), lambda: ortho(m, coefficients=(float("nan"), 0.0, 0.0)),
                 lambda: ortho(m, eps=0.0), lambda: ortho(m, eps=float("nan")), lambda: ortho(m[:, :0]), lambda: ortho(m, coefficients=(1.0, 2.0))):
        with pytest.raises(ValueError):
            call()
