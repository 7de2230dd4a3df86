"""Layer norm and its gradients against plain implementations in 64 bits.

Tolerances are bounds on rounding errors, element by element: half a unit for the rounding to the type (``ULP``); a sum of a row in
fp32 is made of at most 42 additions in a row (32 values of a thread, five shuffles, four and one more) up to 16384 values and
of 128 up to 57344, so that mean and deviation are off by ``DEEP * 2^-24`` of the mean magnitude, relative to the deviation, and what is made of
them by a few times that.
"""
import pytest
import torch

from test_gpu_experts import BF16, FP16, FP32, TINY, ULP, gen, normal, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def norm():
    from flash_sinkhorn_b200.experts import layer_norm
    return layer_norm


def plain(x, w, b, eps):
    x = x.detach().double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    n = (x - m) * r
    return n, r, n * (1 if w is None else w.detach().double()) + (0 if b is None else b.detach().double())


def check(norm, x, w=None, b=None, dy=None, eps=1e-5):
    t = x.dtype
    f = x.shape[-1]
    deep = (42 if f <= 16384 else 128) * 2.0**-24
    leaves = [v.detach().requires_grad_() for v in (x, w, b) if v is not None]
    it = iter(leaves)
    xl, wl, bl = next(it), next(it) if w is not None else None, next(it) if b is not None else None
    n, r, want = plain(x, w, b, eps)
    wd = torch.ones(f, dtype=torch.float64, device=x.device) if w is None else w.double()
    size = x.double().abs().mean(-1, keepdim=True) * r  # mean magnitude relative to the deviation
    off = 4 * deep * (size + n.abs() * (1 + size))  # of n: by the mean, by the deviation
    bound = ULP[t] * want.abs() + TINY[t] + off * wd.abs() + 2.0**-23 * want.abs()
    got = norm(x, w, b, eps=eps)
    assert got.dtype == t and got.shape == x.shape and got.is_contiguous()
    within(got, want, bound)
    if dy is None:
        return
    y = norm(xl, wl, bl, eps=eps)
    assert torch.equal(y, got)
    grads = torch.autograd.grad(y, leaves, dy)
    g = dy.double()
    u = g * wd
    m1, m2 = u.mean(-1, keepdim=True), (u * n).mean(-1, keepdim=True)
    dx = r * (u - m1 - n * m2)
    mag = u.abs().mean(-1, keepdim=True)
    magn = (u * n).abs().mean(-1, keepdim=True)
    err = 4 * deep * r * (u.abs() + mag + n.abs() * magn) * (1 + size) + r * (off * magn + n.abs() * (u.abs() * off).mean(-1, keepdim=True))
    within(grads[0], dx, ULP[t] * dx.abs() + TINY[t] + err)
    # rows are added one after the other by each thread, then the CTAs' sums by eight warps
    rows = x.numel() // f
    adds = (rows / 8 + 64) * 2.0**-24
    flat = lambda v: v.reshape(-1, f)
    i = 1
    for present, value, terms, more in ((w, g * n, (g * n).abs(), g.abs() * off), (b, g, g.abs(), torch.zeros_like(g))):
        if present is None:
            continue
        want = flat(value).sum(0)
        assert grads[i].dtype == present.dtype and grads[i].shape == (f,)
        within(grads[i], want, ULP[present.dtype] * want.abs() + TINY[present.dtype] + adds * flat(terms).sum(0) + flat(more).sum(0))
        i += 1


SHAPES = [(1, 1), (1, 8), (3, 2), (5, 31), (2, 64), (7, 100), (9, 256), (33, 257), (4, 1000), (300, 2048), (2, 2049), (700, 96), (3, 4096),
          (5, 5001), (2, 8192), (3, 16384), (2, 16392), (2, 20001), (1300, 40)]


@pytest.mark.parametrize("rows,f", SHAPES)
@pytest.mark.parametrize("dtype,weights", [(BF16, FP32), (FP16, FP16), (FP32, FP32), (BF16, BF16)])
def test_layer_norm(norm, rows, f, dtype, weights):
    g = gen(rows * 31 + f)
    x = normal(g, rows, f, dtype=dtype) + 0.5
    check(norm, x, (1 + 0.3 * normal(g, f)).to(weights), normal(g, f, dtype=weights), normal(g, rows, f, dtype=dtype))


@pytest.mark.parametrize("has_w,has_b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("f", [384, 501])
def test_without_weight_or_bias(norm, has_w, has_b, f):
    g = gen(f)
    x = normal(g, 65, f, dtype=BF16)
    check(norm, x, normal(g, f) if has_w else None, normal(g, f, dtype=FP32) if has_b else None, normal(g, 65, f, dtype=BF16))


def test_large_mean_and_scales(norm):
    """The deviation is taken from differences: a mean a thousand times larger loses ten bits, not twenty."""
    g = gen(5)
    x = normal(g, 40, 512) + 1000.0
    check(norm, x, None, None, normal(g, 40, 512))
    check(norm, x * 1e-18, None, None, normal(g, 40, 512), eps=0.0)
    check(norm, (normal(g, 40, 512) * 1e4).half(), None, None, normal(g, 40, 512, dtype=FP16))


def test_shapes_and_strides(norm):
    g = gen(8)
    w, b = normal(g, 48), normal(g, 48)
    check(norm, normal(g, 2, 3, 5, 48, dtype=BF16), w, b, normal(g, 2, 3, 5, 48, dtype=BF16))
    check(norm, normal(g, 48, dtype=BF16), w, b, normal(g, 48, dtype=BF16))
    wide = normal(g, 30, 100, dtype=BF16)
    check(norm, wide[:, 1:49], w, b, normal(g, 30, 60, dtype=BF16)[:, 3:51])  # not aligned
    check(norm, wide[::2, 4:52], w[:], b, normal(g, 15, 48, dtype=BF16))
    check(norm, normal(g, 48, 30, dtype=BF16).t(), w, b, normal(g, 1, 48, dtype=BF16).expand(30, 48))
    check(norm, normal(g, 4, 7, 96, dtype=FP32)[:, 2:5, :48], w, b, normal(g, 4, 3, 48))
    check(norm, normal(g, 30, 48, dtype=BF16), normal(g, 96)[::2], normal(g, 97)[1:49], normal(g, 30, 48, dtype=BF16))


def test_constant_rows_and_rows_that_are_not_finite(norm):
    x = torch.full((4, 64), 3.0, device="cuda")
    y = norm(x, None, torch.full((64,), 2.0, device="cuda"))
    assert torch.equal(y, torch.full_like(x, 2.0))
    x = normal(gen(1), 6, 200)
    ref = norm(x)
    x[1, 3], x[4, 199] = float("nan"), float("inf")
    y = norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all()
    assert torch.equal(y[[0, 2, 3, 5]], ref[[0, 2, 3, 5]])


def test_gradients_against_differences(norm):
    g = gen(3)
    x, w, b, dy = normal(g, 3, 10), 1 + 0.2 * normal(g, 10), normal(g, 10), normal(g, 3, 10)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    grads = torch.autograd.grad(norm(*leaves), leaves, dy)
    for i, leaf in enumerate((x, w, b)):
        for j in range(leaf.numel()):
            values = []
            for h in (2.0**-7, -(2.0**-7)):
                moved = [v.double() for v in (x, w, b)]
                moved[i] = moved[i].clone()
                moved[i].view(-1)[j] += h
                values.append((plain(*moved, 1e-5)[2] * dy.double()).sum().item())
            slope = (values[0] - values[1]) / 2.0**-6
            assert abs(grads[i].reshape(-1)[j].item() - slope) < 2e-3 * (1 + abs(slope))  # third derivatives of order 1 to 30, times h^2 / 6


def test_only_some_gradients(norm):
    g = gen(4)
    x, w, b, dy = normal(g, 50, 72), normal(g, 72), normal(g, 72), normal(g, 50, 72)
    full = [v.clone().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(norm(*full), full, dy)
    for i in range(3):
        leaves = [v.clone().requires_grad_(j == i) for j, v in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(norm(*leaves), [leaves[i]], dy)
        assert torch.equal(got, want[i])


def test_empty(norm):
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = norm(x, w)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros(32, device="cuda")) and x.grad.shape == (0, 32)
    assert norm(torch.zeros(2, 0, 8, device="cuda")).shape == (2, 0, 8)


def test_same_bits_on_another_stream_and_in_a_graph(norm):
    g = gen(9)
    x, w, b, dy = normal(g, 513, 1024, dtype=BF16), normal(g, 1024), normal(g, 1024), normal(g, 513, 1024, dtype=BF16)

    def step(x, w, b):
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        y = norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(want, again))
    with torch.cuda.stream(side):
        step(x, w, b)
    torch.cuda.synchronize()
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, w, b)
    for seed in (1, 2):
        static.copy_(normal(gen(seed), 513, 1024, dtype=BF16))
        graph.replay()
        fresh = step(static, w, b)
        assert all(torch.equal(u, v) for u, v in zip(out, fresh))


def test_refusals(norm):
    x, w = torch.zeros(4, 8, device="cuda", dtype=BF16), torch.zeros(8, device="cuda")
    for call in (lambda: norm(x.double()), lambda: norm(x, w[:4]), lambda: norm(x, w.half()), lambda: norm(x, w, w.bfloat16()),
                 lambda: norm(x, w.cpu()), lambda: norm(x.cpu()), lambda: norm(x, eps=-1.0), lambda: norm(x, eps=float("nan")),
                 lambda: norm(x[:, :0]), lambda: norm(x[0, 0]), lambda: norm(x, w.view(1, 8))):
        with pytest.raises(ValueError):
            call()
