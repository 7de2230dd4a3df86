"""Products in 8-bit floating point against plain implementations in 64 bits.

The codes are defined exactly (scales are powers of two), so the products are compared with those of the rounded operands. Bounds: half a unit
for the rounding to the type, and 2^-15 of the sum of the products' magnitudes for the sums: within a block of 128 the tensor core adds
in fp32 with a bit or two less than IEEE addition (128 * 2^-23), the blocks' sums are scaled and added in fp32 (2^-24 each, at most 64 blocks).
"""
import pytest
import torch

from test_gpu_experts import BF16, FP16, FP32, TINY, ULP, gen, normal, within

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ex():
    from flash_sinkhorn_b200 import experts
    return experts


def scale_of(top):
    """Smallest power of two from 2^-126 on by which `top` [..] is at most 448; NaN for what is not finite."""
    top = top.double()
    s = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0**-140) / 448)))
    s = torch.where(top > 448 * s, 2 * s, torch.where(top <= 448 * (s / 2), s / 2, s)).clamp_min(2.0**-126)
    return torch.where(torch.isfinite(top), s, float("nan"))


def rounded(v):
    """The nearest values of the 8-bit type, ties to even, for magnitudes up to 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def rows8(x):
    """What rows stand for in 8 bits."""
    out = x.detach().double().clone()
    for at in range(0, x.shape[1], 128):
        b = out[:, at:at + 128]
        s = scale_of(b.abs().amax(1, keepdim=True))
        out[:, at:at + 128] = rounded(b / s) * s
    return out


def blocks8(w):
    """Codes' values and scales of weights [E, N, K]."""
    e, n, k = w.shape
    v = w.detach().double().clone()
    scales = torch.zeros(e, -(-n // 128), -(-k // 128), dtype=torch.float64, device=w.device)
    for i in range(0, n, 128):
        for j in range(0, k, 128):
            b = v[:, i:i + 128, j:j + 128]
            s = scale_of(b.abs().amax((1, 2)))
            scales[:, i // 128, j // 128] = s
            v[:, i:i + 128, j:j + 128] = rounded(b / s[:, None, None])
    return v, scales


def wide(scales, n, k):
    return scales.double().repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]


def grouped(x, w, ends, transposed=False):
    """Products in 64 bits and the sums of their magnitudes; zeros for rows of no group."""
    n = w.shape[2] if transposed else w.shape[1]
    y = torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    lo = 0
    for e, hi in enumerate(ends):
        hi = max(lo, min(hi, x.shape[0]))
        m = w[e] if transposed else w[e].T
        y[lo:hi] = x[lo:hi] @ m
        size[lo:hi] = x[lo:hi].abs() @ m.abs()
        lo = hi
    return y, size


def offsets_of(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def close(got, want, size, t):
    within(got, want, ULP[t] * want.abs() + TINY[t] + 2.0**-15 * size)


@pytest.mark.parametrize("e,n,k", [(1, 1, 1), (2, 128, 128), (3, 130, 257), (1, 300, 501), (4, 64, 1000), (2, 257, 16)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_to_blocks8(ex, e, n, k, dtype):
    g = gen(n + k)
    w = (normal(g, e, n, k) * torch.exp(3 * normal(g, e, n, k))).to(dtype)
    q = ex.to_blocks8(w)
    codes, scales = blocks8(w)
    assert q.codes.dtype == E4M3 and q.codes.shape == w.shape and q.scales.shape == scales.shape and q.codes.stride(1) % 16 == 0
    fine = torch.isfinite(wide(scales, n, k))  # fp16 weights this large are infinite here and there
    within(q.scales, scales, torch.zeros_like(scales))
    assert torch.equal(q.codes.double(), torch.where(fine, codes, 0.0))
    off = (q.codes.double() * wide(q.scales, n, k) - w.double()).abs()
    assert (off <= torch.maximum(w.double().abs() / 16, wide(q.scales, n, k) * 2.0**-10))[fine].all()


def test_to_blocks8_borders(ex):
    """Largest magnitudes next to the powers of two at which the scale changes, ties, zeros, the smallest and largest values, NaN."""
    tops = [448.0, 449.0, 447.0, 450.0, 448.0 * 2**20, 452.0 * 2**20, 1.75, 1.7578125, 3.0e38, 1e-38, 0.0, float("inf"), float("nan"), 2.0**-126, 416.0]
    w = torch.zeros(len(tops), 3, 40, device="cuda", dtype=BF16)
    w[:, 1] = torch.linspace(-1, 1, 40, device="cuda").bfloat16()
    t = torch.tensor(tops, device="cuda").bfloat16()
    finite = torch.isfinite(t)
    w[:, 1] = torch.where(finite[:, None], w[:, 1].float() * t[:, None].float(), w[:, 1].float()).bfloat16()
    w[:, 2, 5] = t
    q = ex.to_blocks8(w)
    codes, scales = blocks8(w)
    within(q.scales, scales, torch.zeros_like(scales))
    assert torch.equal(q.codes.double()[finite], codes[finite])
    assert torch.isnan(q.scales[~finite]).all() and (q.codes.double()[~finite] == 0).all()


def test_to_blocks8_strides(ex):
    g = gen(2)
    for w in (normal(g, 3, 50, 70, dtype=BF16)[:, :, 3:40], normal(g, 3, 70, 50, dtype=BF16).transpose(1, 2), normal(g, 1, 50, 70, dtype=BF16).expand(3, 50, 70),
              normal(g, 6, 50, 64, dtype=FP16)[::2, ::3]):
        q, p = ex.to_blocks8(w), ex.to_blocks8(w.contiguous().clone())
        assert torch.equal(q.codes.float(), p.codes.float()) and torch.equal(q.scales, p.scales)


COUNTS = [([1], 40, 64), ([2], 100, 300), ([1, 0, 1], 257, 130), ([0, 1], 64, 16), ([3], 8, 8), ([0, 3, 5], 33, 129), ([7, 0, 1, 64], 300, 501),
          ([128, 1, 127], 128, 128), ([129, 300], 256, 384), ([40, 200, 0, 33, 1], 520, 1000), ([0, 0, 5], 1, 1), ([513], 65, 2048), ([2], 2048, 8320)]


@pytest.mark.parametrize("counts,n,k", COUNTS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("spare", [0, 3])
def test_grouped_mm8(ex, counts, n, k, dtype, spare):
    """Rows in order; `spare` rows of no expert behind them."""
    g = gen(sum(counts) + n)
    x = (normal(g, sum(counts) + spare, k) * torch.exp(normal(g, sum(counts) + spare, k))).to(dtype)
    w = normal(g, len(counts), n, k, scale=k**-0.5, dtype=dtype)
    off = offsets_of(counts)
    q = ex.to_blocks8(w)
    got = ex.grouped_mm8(x, q, off)
    want, size = grouped(rows8(x), q.codes.double() * wide(q.scales, n, k), off[1:].tolist())
    assert got.dtype == dtype
    close(got, want, size, dtype)
    assert torch.equal(ex.grouped_mm8(x, w, off), got)  # weights put into 8 bits in the call


def routed(ex, g, t, k, e, off=0.2):
    mask = torch.rand(t, generator=g, device="cuda") >= off
    return ex.route_tokens(normal(g, t, e), k, mask=mask)


@pytest.mark.parametrize("t,slots,e,n,k", [(1, 1, 4, 64, 64), (1, 2, 8, 300, 256), (2, 1, 3, 130, 501), (5, 2, 4, 96, 130), (37, 4, 16, 257, 300),
                                           (500, 2, 3, 300, 520), (900, 4, 8, 512, 384), (6000, 2, 2, 600, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gathered_rows_and_gradients(ex, t, slots, e, n, k, dtype):
    g = gen(t + n)
    r = routed(ex, g, t, slots, e)
    x = normal(g, t, k, dtype=dtype).requires_grad_()
    w = normal(g, e, n, k, scale=k**-0.5, dtype=dtype).requires_grad_()
    dy = normal(g, t * slots, n, dtype=dtype)
    y = ex.grouped_mm8(x, w, r, gather=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    codes, scales = blocks8(w)
    v, ends = codes * wide(scales, n, k), r.offsets[1:].tolist()
    live = (r.rows >= 0)[:, None]
    from_rows = r.rows.long().clamp_min(0)
    want, size = grouped(rows8(x)[from_rows] * live, v, ends)
    close(y, want, size, dtype)
    want, size = grouped(rows8(dy), v, ends, transposed=True)
    back = torch.zeros(t, k, dtype=torch.float64, device="cuda").index_add_(0, from_rows, want * live)
    size = torch.zeros_like(back).index_add_(0, from_rows, size * live)
    close(dx, back, size, dtype)
    lo = 0
    for i, hi in enumerate(ends):  # the 16-bit product of what was given
        a, b = dy[lo:hi].double(), x.detach().double()[from_rows[lo:hi]]
        close(dw[i], a.T @ b, a.abs().T @ b.abs() * max(1.0, (hi - lo) / 128), dtype)
        lo = hi
    # held weights: the same result and gradient to x
    xq = x.detach().requires_grad_()
    yq = ex.grouped_mm8(xq, ex.to_blocks8(w.detach()), r, gather=True)
    assert torch.equal(yq, y)
    assert torch.equal(torch.autograd.grad(yq, xq, dy)[0], dx)
    # one gradient alone
    x1 = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ex.grouped_mm8(x1, w.detach(), r, gather=True), x1, dy)[0], dx)
    w1 = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ex.grouped_mm8(x.detach(), w1, r, gather=True), w1, dy)[0], dw)


@pytest.mark.parametrize("counts,n,k", [([1], 40, 64), ([3, 0, 5], 300, 129), ([600, 700], 384, 520), ([3000], 300, 640)])
def test_gradients_in_order(ex, counts, n, k):
    g = gen(n)
    x, w = normal(g, sum(counts) + 2, k, dtype=BF16).requires_grad_(), normal(g, len(counts), n, k, dtype=BF16).requires_grad_()
    dy = normal(g, sum(counts) + 2, n, dtype=BF16)
    off = offsets_of(counts)
    dx, dw = torch.autograd.grad(ex.grouped_mm8(x, w, off), (x, w), dy)
    codes, scales = blocks8(w)
    want, size = grouped(rows8(dy), codes * wide(scales, n, k), off[1:].tolist(), transposed=True)
    close(dx, want, size, BF16)
    assert torch.equal(dw, torch.autograd.grad(ex.grouped_mm(x, w, off), w, dy)[0])


def test_gradient_against_differences(ex):
    """Where nothing is rounded (small whole numbers), the gradients are those of the product itself."""
    g = gen(1)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").to(BF16)
    x, w, dy = whole(5, 12), whole(2, 9, 12), whole(5, 9)
    off = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    grads = torch.autograd.grad(ex.grouped_mm8(leaves[0], leaves[1], off), leaves, dy)
    value = lambda x, w: (grouped(x.double(), w.double(), [2, 5])[0] * dy.double()).sum().item()
    for i, leaf in enumerate((x, w)):
        for j in range(0, leaf.numel(), 7):
            moved = [x.clone(), w.clone()]
            moved[i].view(-1)[j] += 1
            up = value(*moved)
            moved[i].view(-1)[j] -= 2
            assert grads[i].reshape(-1)[j].item() == (up - value(*moved)) / 2


def test_scales_of_any_value_and_strides(ex):
    g = gen(6)
    e, n, k = 3, 200, 260
    store = normal(g, e, n + 3, 300).clamp(-3, 3).to(E4M3)
    scales = torch.rand(e, 2, 3, generator=g, device="cuda") + 0.1
    off = offsets_of([5, 0, 40])
    wide_x = normal(g, 45, 300, dtype=BF16)
    for codes in (store[:, :n, :k], store[:, 1:n + 1, 7:k + 7], store[:, :n, :k].transpose(1, 2).contiguous().transpose(1, 2)):
        for x in (wide_x[:, :k], wide_x[:, 5:k + 5], normal(g, k, 45, dtype=BF16).t()):
            want, size = grouped(rows8(x), codes.double() * wide(scales, n, k), off[1:].tolist())
            close(ex.grouped_mm8(x, ex.Blocks8(codes, scales), off), want, size, BF16)


@pytest.mark.parametrize("counts", [[1, 1], [3, 2, 5], [200, 100, 300]])
def test_values_that_are_not_finite_stay_in_their_rows_and_blocks(ex, counts):
    g = gen(7)
    n, k = 300, 400
    x, w = normal(g, sum(counts), k, dtype=BF16), normal(g, len(counts), n, k, dtype=BF16)
    off = offsets_of(counts)
    ref = ex.grouped_mm8(x, w, off)
    bad = x.clone()
    bad[1, 390] = float("inf")
    y = ex.grouped_mm8(bad, w, off)
    assert torch.isnan(y[1]).all()
    keep = [i for i in range(sum(counts)) if i != 1]
    assert torch.equal(y[keep], ref[keep])
    w = w.clone()
    w[1, 130, 5] = float("nan")
    y = ex.grouped_mm8(x, w, off)
    lo, hi = counts[0], counts[0] + counts[1]
    assert torch.isnan(y[lo:hi, 128:256]).all()
    y[lo:hi, 128:256] = ref[lo:hi, 128:256]
    assert torch.equal(y, ref)


def test_offsets_and_row_numbers_outside(ex):
    g = gen(8)
    x, w = normal(g, 40, 64, dtype=BF16), normal(g, 3, 96, 64, dtype=BF16)
    ref = lambda ends: grouped(rows8(x), blocks8(w)[0] * wide(blocks8(w)[1], 96, 64), ends)
    for given, ends in (([0, 10, 5, 60], [10, 10, 40]), ([7, -3, 20, 30], [0, 20, 30]), ([0, 40, 40, 40], [40, 40, 40]), ([0, 0, 0, 0], [0, 0, 0])):
        close(ex.grouped_mm8(x, w, torch.tensor(given, dtype=torch.int32, device="cuda")), *ref(ends), BF16)
    r = routed(ex, g, 40, 2, 3, off=0.0)
    rows = r.rows.clone()
    rows[3], rows[9], rows[11] = 40, -5, 2**31 - 1
    y = ex.grouped_mm8(x, w, r._replace(rows=rows), gather=True)
    want = ex.grouped_mm8(x, w, r, gather=True)
    want[[3, 9, 11]] = 0
    assert torch.equal(y, want)


def test_zero_rows(ex):
    w = normal(gen(1), 2, 48, 32, dtype=BF16)
    x = torch.zeros(0, 32, device="cuda", dtype=BF16, requires_grad=True)
    wl = w.requires_grad_()
    y = ex.grouped_mm8(x, wl, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert y.shape == (0, 48)
    y.sum().backward()
    assert x.grad.shape == (0, 32) and torch.equal(wl.grad, torch.zeros_like(w))


def test_expert_mlp_with_held_weights(ex):
    g = gen(11)
    t, d, f, e, k = 70, 96, 136, 5, 2
    r0 = routed(ex, g, t, k, e)
    x = normal(g, t, d, dtype=BF16)
    w_in, w_out = (ex.to_blocks8(normal(g, *s, scale=s[2]**-0.5, dtype=BF16)) for s in ((e, 2 * f, d), (e, d, f)))
    xl, gates = x.clone().requires_grad_(), r0.gates.detach().clone().requires_grad_()
    r = r0._replace(gates=gates)
    y = ex.expert_mlp(xl, w_in, w_out, r)
    h = ex.gated_act(ex.grouped_mm8(x, w_in, r0, gather=True), r0)
    want = ex.combine_rows(ex.grouped_mm8(h, w_out, r0), r0, weighted=False)
    assert torch.equal(y, want) and torch.equal(ex.expert_mlp(x, w_in, w_out, r0), want)
    dx, dgates = torch.autograd.grad(y, (xl, gates), normal(g, t, d, dtype=BF16))
    assert torch.isfinite(dx).all() and dx.abs().sum() > 0 and dgates.abs().sum() > 0
    with pytest.raises(ValueError):
        ex.expert_mlp(x, w_in, normal(g, e, d, f, dtype=BF16), r)


@pytest.mark.parametrize("t", [1, 300])
def test_same_bits_on_another_stream_and_in_a_graph(ex, t):
    g = gen(12)
    e, n, k = 6, 384, 512
    r = routed(ex, g, t, 2, e, off=0.0)
    w, dy = normal(g, e, n, k, dtype=BF16), normal(g, 2 * t, n, dtype=BF16)

    def step(x):
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = ex.grouped_mm8(leaves[0], leaves[1], r, gather=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    x = normal(g, t, k, dtype=BF16)
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x)
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(want, again))
    torch.cuda.synchronize()
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in (1, 2):
        static.copy_(normal(gen(seed), t, k, dtype=BF16))
        graph.replay()
        assert all(torch.equal(u, v) for u, v in zip(out, step(static)))


@pytest.mark.parametrize("counts,n,k", [([5, 9], 200, 256), ([900, 800, 2000, 3000, 10, 700], 2048, 256)])
def test_products_that_give_up(ex, counts, n, k):
    """With no clocks to wait the result is NaN and the health word says so; afterwards all is as before."""
    from flash_sinkhorn_b200 import _lib
    lib = _lib.load()
    g = gen(13)
    x, w, off = normal(g, sum(counts), k, dtype=BF16), ex.to_blocks8(normal(g, len(counts), n, k, dtype=BF16)), offsets_of(counts)
    want = ex.grouped_mm8(x, w, off)
    assert lib.fs_device_error() == 0
    before = lib.fs_set_product_limit(0)
    try:
        y = ex.grouped_mm8(x, w, off)
    finally:
        lib.fs_set_product_limit(before)
    assert torch.isnan(y).all() and lib.fs_device_error() == 1
    assert lib.fs_clear_device_error() == 0 and lib.fs_device_error() == 0
    assert torch.equal(ex.grouped_mm8(x, w, off), want)


def test_refusals(ex):
    w, x = torch.zeros(2, 8, 16, device="cuda", dtype=BF16), torch.zeros(6, 16, device="cuda", dtype=BF16)
    q, off = ex.to_blocks8(w), torch.zeros(3, dtype=torch.int32, device="cuda")
    calls = [lambda: ex.to_blocks8(w[0]), lambda: ex.to_blocks8(w.float()), lambda: ex.to_blocks8(w.cpu()), lambda: ex.to_blocks8(w[:, :0]),
             lambda: ex.grouped_mm8(x, w.half(), off), lambda: ex.grouped_mm8(x.float(), q, off), lambda: ex.grouped_mm8(x[:, :8], q, off),
             lambda: ex.grouped_mm8(x, q, off[:2]), lambda: ex.grouped_mm8(x, q, off.long()), lambda: ex.grouped_mm8(x, q, off.cpu()),
             lambda: ex.grouped_mm8(x, q, off, gather=True), lambda: ex.grouped_mm8(x, ex.Blocks8(q.codes, q.scales[:1]), off),
             lambda: ex.grouped_mm8(x, ex.Blocks8(q.codes, q.scales.double()), off), lambda: ex.grouped_mm8(x, ex.Blocks8(w, q.scales), off),
             lambda: ex.grouped_mm8(x, ex.Blocks8(q.codes.cpu(), q.scales), off), lambda: ex.grouped_mm8(x, ex.Blocks8(q.codes, q.scales.cpu()), off),
             lambda: ex.grouped_mm8(x.cpu(), q, off)]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    y = ex.grouped_mm8(x.requires_grad_(), q, off)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
