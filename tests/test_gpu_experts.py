"""Operators of routed experts against plain implementations in 64 bits.

Tolerances are bounds on the rounding errors of the definition, element by element: half a unit in the last place for
each rounding to the type (``ULP``), and for sums of n terms in fp32 an error of at most 2^-22 of the sum of the terms'
magnitudes for each term (a tensor core adds with one or two bits less than IEEE addition).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ULP = {BF16: 2.0**-8, FP16: 2.0**-11, FP32: 2.0**-24}  # relative, half a unit
TINY = {BF16: 2.0**-130, FP16: 2.0**-25, FP32: 2.0**-130}  # absolute, where the type runs out of exponents
ACC = 2.0**-22
FUN = 2.0**-19  # relative error of sigmoid and of the few products around it in fp32


class Kernels:
    """The public operators, and the kernels by themselves (leading underscore)."""

    def __init__(self):
        from flash_sinkhorn_b200 import _lib, experts
        self.__dict__.update({name: getattr(experts, name) for name in experts.__all__})
        raw = _lib.torch_binding()
        self._mm = lambda x, rows, count, w, offsets, transposed=False, dtype=None: raw.mm(x, rows, count, w, offsets, transposed,
                                                                                          dtype == FP32)
        self._wgrad, self._gather, self._act, self._act_grad = raw.wgrad, raw.gather, raw.act, raw.act_grad


@pytest.fixture(scope="module")
def ex():
    return Kernels()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, scale=1.0, dtype=FP32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound):
    """|got - want| <= bound everywhere, infinities and NaN in the same places."""
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
    over = ((got - want).abs() - bound)[~odd]
    assert over.numel() == 0 or over.max() <= 0, f"off by {over.max().item():.3g} more than allowed"


# ---------------------------------------------------------------------------------------------------------------
# Routing
# ---------------------------------------------------------------------------------------------------------------


def plain_route(logits, k, bias, mask, over_all):
    """Everything of a Routing, the gates in 64 bits; one token after the other, on the host."""
    l = logits.detach().float().cpu()
    b = torch.zeros(l.shape[1]) if bias is None else bias.float().cpu()
    t, e = l.shape
    on = (l != -math.inf) & (b != -math.inf)
    if mask is not None:
        on &= mask.cpu()[:, None]
    score = l + b
    experts = torch.full((t, k), -1, dtype=torch.int32)
    gates = torch.zeros(t, k, dtype=torch.float64)
    for i in range(t):
        live = [j for j in range(e) if on[i, j]]
        s = score[i].tolist()
        live.sort(key=lambda j: (0 if s[j] != s[j] else 1, -s[j] if s[j] == s[j] else 0.0, j))
        chosen = live[:k]
        experts[i, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        if chosen:
            over = sorted(live) if over_all else chosen
            z = l[i, over].double()
            top = z[~torch.isnan(z)].max() if (~torch.isnan(z)).any() else torch.tensor(math.nan)
            gates[i, :len(chosen)] = torch.exp(l[i, chosen].double() - top) / torch.exp(z - top).sum()
    flat = experts.reshape(-1)
    order = [p for j in range(e) for p in (flat == j).nonzero()[:, 0].tolist()]
    pairs = torch.full((t * k,), -1, dtype=torch.int32)
    pairs[:len(order)] = torch.tensor(order, dtype=torch.int32)
    position = torch.full((t * k,), -1, dtype=torch.int32)
    position[torch.tensor(order, dtype=torch.int64)] = torch.arange(len(order), dtype=torch.int32)
    counts = torch.tensor([0] + [int((flat == j).sum()) for j in range(e)])
    rows = torch.where(pairs >= 0, pairs // k, -1)
    return gates, experts, counts.cumsum(0).int(), pairs, rows, position.reshape(t, k)


def check_route(ex, logits, k, bias=None, mask=None, over_all=False):
    got = ex.route_tokens(logits, k, bias=bias, mask=mask, normalize="all" if over_all else "selected")
    want = plain_route(logits, k, bias, mask, over_all)
    for name, g, w in zip(ex.Routing._fields[1:], got[1:], want[1:]):
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), w), name
    # exp and a quotient of a sum of up to 1024 terms, adds in fp32
    within(got.gates.cpu(), want[0], 2.0**-20 * want[0].abs() + 1e-40)
    return got


@pytest.mark.parametrize("t,e,k", [(0, 4, 2), (1, 1, 1), (1, 64, 4), (31, 5, 5), (33, 33, 3), (256, 64, 8), (257, 64, 8),
                                   (700, 31, 1), (900, 128, 8), (300, 300, 6), (61, 1024, 32), (5000, 7, 2)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_route(ex, t, e, k, dtype):
    g = gen(t * 7 + e)
    logits = normal(g, t, e, dtype=dtype)
    check_route(ex, logits, k, over_all=bool(t % 2))
    check_route(ex, logits, k, bias=normal(g, e), mask=torch.rand(t, generator=g, device="cuda") < 0.7, over_all=not t % 2)


def test_route_ties_go_to_the_lower_expert_and_zeros_tie(ex):
    g = gen(3)
    logits = torch.randint(-2, 3, (400, 96), generator=g, device="cuda").float() * 0.5
    logits[logits == 0] *= torch.where(torch.rand(int((logits == 0).sum()), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    check_route(ex, logits, 7)
    check_route(ex, torch.full((50, 40), torch.finfo(FP32).min, device="cuda"), 3, over_all=True)  # lowest is a value


@pytest.mark.parametrize("over_all", [False, True])
def test_route_of_experts_that_are_off(ex, over_all):
    g = gen(4)
    logits = normal(g, 200, 20)
    logits[torch.rand(200, 20, generator=g, device="cuda") < 0.8] = -math.inf  # some rows keep fewer than k, some none
    logits[5] = -math.inf
    bias = normal(g, 20)
    bias[[3, 7]] = -math.inf
    logits[:, 3] = math.nan  # under a bias of -inf it does not show
    mask = torch.arange(200, device="cuda") % 9 != 0
    logits[9] = math.inf  # masked
    r = check_route(ex, logits, 4, bias=bias, mask=mask, over_all=over_all)
    assert torch.isfinite(r.gates).all() and (r.experts[5] == -1).all() and (r.gates[9] == 0).all()
    none = check_route(ex, logits, 4, bias=bias, mask=torch.zeros_like(mask))
    assert int(none.offsets[-1]) == 0


def test_route_infinite_and_nan_logits_show(ex):
    logits = torch.zeros(4, 8, device="cuda")
    logits[0, 6] = math.nan
    logits[1, 2] = math.inf
    logits[2, 1] = 3e38
    r = ex.route_tokens(logits, 2, bias=torch.full((8,), 3e38, device="cuda"))
    assert r.experts.tolist() == [[6, 0], [2, 0], [1, 0], [0, 1]]
    assert torch.isnan(r.gates[0]).all() and torch.isnan(r.gates[1]).any()
    assert r.gates[2].tolist() == [1.0, 0.0] and r.gates[3].tolist() == [0.5, 0.5]


def test_route_strided_logits(ex):
    wide = normal(gen(5), 300, 200)
    check_route(ex, wide[:, 11:75], 3)
    check_route(ex, wide.t()[:64, :], 3)
    check_route(ex, wide[::2, :40], 3)
    check_route(ex, wide[:1, :40].expand(70, 40), 3)


def test_route_of_a_large_batch(ex):
    """More tokens than one round of all CTAs, against torch's stable sorts."""
    t, e, k = 150_001, 48, 6
    logits = normal(gen(6), t, e)
    r = ex.route_tokens(logits, k)
    chosen = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.experts.long(), chosen)
    order = torch.sort(chosen.reshape(-1), stable=True).indices
    assert torch.equal(r.pairs.long(), order) and torch.equal(r.rows.long(), order // k)
    assert torch.equal(r.position.reshape(-1).long()[order], torch.arange(t * k, device="cuda"))
    assert torch.equal(r.offsets.long(), torch.cat([order.new_zeros(1), chosen.reshape(-1).bincount(minlength=e).cumsum(0)]))


@pytest.mark.parametrize("over_all", [False, True])
@pytest.mark.parametrize("dtype,e,k", [(FP32, 40, 5), (BF16, 128, 8), (FP16, 600, 2), (FP32, 3, 3)])
def test_route_gradient(ex, over_all, dtype, e, k):
    g = gen(e)
    t = 150
    logits = normal(g, t, e, dtype=dtype)
    logits[torch.rand(t, e, generator=g, device="cuda") < 0.3] = -math.inf
    logits[4] = -math.inf
    mask = torch.rand(t, generator=g, device="cuda") < 0.9
    logits.requires_grad_(True)
    r = ex.route_tokens(logits, k, mask=mask, normalize="all" if over_all else "selected")
    w = normal(g, t, k)
    (got,) = torch.autograd.grad(r.gates, (logits,), w)
    assert got.dtype == dtype

    z = logits.detach().double()
    on = torch.isfinite(z) & mask[:, None]
    chosen, taken = r.experts.long().clamp_min(0), r.experts >= 0
    zz = z.masked_fill(~on, -1e300).requires_grad_(True)
    if over_all:
        gates = torch.softmax(zz, 1).gather(1, chosen)
    else:
        gates = torch.softmax(zz.gather(1, chosen).masked_fill(~taken, -math.inf), 1)
    (want,) = torch.autograd.grad((gates.masked_fill(~taken, 0.0) * w.double()).sum(), (zz,))
    want = torch.nan_to_num(want).masked_fill(~on, 0.0)
    size = w.abs().double().sum(1, keepdim=True)
    within(got, want, ULP[dtype] * want.abs() + 2.0**-19 * size + TINY[dtype])


def test_route_gradient_against_differences(ex):
    g = gen(12)
    logits, w = normal(g, 40, 12), normal(g, 40, 4)
    d = normal(g, 40, 12)
    for over in ("selected", "all"):
        leaf = logits.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(ex.route_tokens(leaf, 4, normalize=over).gates, (leaf,), w)
        h = 2.0**-9
        fixed = ex.route_tokens(logits, 4).experts.long()
        up = (ex.route_tokens(logits + h * d, 4, normalize=over), ex.route_tokens(logits - h * d, 4, normalize=over))
        # tokens whose choice the step does not change
        same = (up[0].experts.long() == fixed).all(1) & (up[1].experts.long() == fixed).all(1)
        diff = ((up[0].gates - up[1].gates) * w).sum(1) / (2 * h)
        # third-order remainder h^2 |d|^3 and fp32 noise 2^-22 / h
        err = (diff - (grad * d).sum(1)).abs()[same]
        assert int(same.sum()) > 20 and err.max() < h * h * 30 * w.abs().sum(1).max() + 2.0**-20 / h * w.abs().sum(1).max()


# ---------------------------------------------------------------------------------------------------------------
# Grouped products
# ---------------------------------------------------------------------------------------------------------------


def offsets_of(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(dtype=torch.int32, device="cuda")


def group_rows(offsets, r):
    ends = offsets.tolist()
    return [(max(0, lo), min(r, hi)) for lo, hi in zip(ends[:-1], ends[1:])]


def check_mm(ex, x, w, offsets, rows=None):
    """Forward and both gradients of plain groups (rows None), or of rows gathered from x, through the private calls."""
    r = x.shape[0] if rows is None else rows.shape[0]
    n, k = w.shape[1:]
    dtype = x.dtype
    got = ex._mm(x, rows, r, w, offsets)
    xs = x.double() if rows is None else x.double()[rows.long().clamp_min(0)]
    want, size = torch.zeros(r, n, dtype=torch.float64, device="cuda"), torch.zeros(r, n, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(group_rows(offsets, r)):
        if hi > lo:
            want[lo:hi] = xs[lo:hi] @ w[e].double().T
            size[lo:hi] = xs[lo:hi].abs() @ w[e].double().abs().T
    within(got, want, ULP[dtype] * want.abs() + ACC * size * min(k, 64) + TINY[dtype])
    return got


def check_wgrad(ex, dy, x, offsets):
    e, n, k, r, dtype = offsets.shape[0] - 1, dy.shape[1], x.shape[1], x.shape[0], x.dtype
    got = ex._wgrad(dy, x, offsets)
    ys, xs = dy.double(), x.double()
    want, size = torch.zeros(e, n, k, dtype=torch.float64, device="cuda"), torch.zeros(e, n, k, dtype=torch.float64, device="cuda")
    most = 1
    for j, (lo, hi) in enumerate(group_rows(offsets, r)):
        if hi > lo:
            want[j] = ys[lo:hi].T @ xs[lo:hi]
            size[j] = ys[lo:hi].abs().T @ xs[lo:hi].abs()
            most = max(most, hi - lo)
    within(got, want, ULP[dtype] * want.abs() + ACC * size * min(most, 64) + TINY[dtype])
    return got


GROUPS = [
    [0, 1, 0, 2, 15, 16, 17, 0],
    [127, 128, 129, 1],
    [255, 0, 256, 257],
    [1],
    [0, 0, 0],
    [3] * 40,
    [700, 5],
    [31, 33, 63, 64, 65],
]


@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: "-".join(map(str, c[:5])))
@pytest.mark.parametrize("n,k", [(64, 64), (256, 128), (100, 72), (65, 33), (1, 1), (300, 300), (129, 520), (8, 1000)])
def test_grouped_mm(ex, counts, n, k):
    dtype = BF16 if (n + k) % 3 else FP16
    g = gen(n * 131 + k)
    r = sum(counts) + 3  # three rows of no expert
    off = offsets_of(counts)
    x, w = normal(g, r, k, dtype=dtype), normal(g, len(counts), n, k, scale=k**-0.5, dtype=dtype)
    dy = normal(g, r, n, dtype=dtype)
    assert (check_mm(ex, x, w, off)[sum(counts):] == 0).all()
    check_mm(ex, dy, w.transpose(1, 2), off)
    check_wgrad(ex, dy, x, off)


@pytest.mark.parametrize("k,n,tokens,slots,e", [(64, 96, 1, 2, 16), (256, 192, 5, 1, 3), (136, 72, 33, 4, 64), (300, 501, 200, 2, 7),
                                                (512, 320, 700, 6, 12), (1024, 256, 64, 8, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_grouped_mm_of_gathered_rows(ex, k, n, tokens, slots, e, dtype):
    g = gen(k + n)
    logits = normal(g, tokens, e)
    mask = torch.arange(tokens, device="cuda") % 7 != 3
    routing = ex.route_tokens(logits, slots, mask=mask)
    x, w = normal(g, tokens, k, dtype=dtype), normal(g, e, n, k, scale=k**-0.5, dtype=dtype)
    r = tokens * slots
    check_mm(ex, x, w, routing.offsets, routing.rows)
    dy = normal(g, r, n, dtype=dtype)
    xs = ex._gather(x, routing.rows)
    live = routing.rows >= 0
    assert torch.equal(xs[live], x[routing.rows[live].long()]) and not xs[~live].any()
    check_wgrad(ex, dy, xs, routing.offsets)
    dyt = normal(g, tokens, n, dtype=dtype)
    check_mm(ex, dyt, w.transpose(1, 2), routing.offsets, routing.rows)

    # through the public call: the gradient of a token is the sum over its rows in fp32, rounded once
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = ex.grouped_mm(xl, wl, routing, gather=True)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy)
    assert torch.equal(y, ex._mm(x, routing.rows, r, w, routing.offsets))
    assert torch.equal(dw, ex._wgrad(dy, xs, routing.offsets))
    pos = routing.position.long()
    part = ex._mm(dy, None, r, w, routing.offsets, transposed=True, dtype=FP32).double()[pos.clamp_min(0)] * (pos >= 0)[..., None]
    within(dx, part.sum(1), ULP[dtype] * part.sum(1).abs() + ACC * part.abs().sum(1) + TINY[dtype])


@pytest.mark.parametrize("counts,n,k", [([300, 0, 500, 200], 384, 512), ([5000, 300, 2000], 256, 1024), ([2] * 90, 1024, 768)])
def test_grouped_mm_larger(ex, counts, n, k):
    g = gen(k)
    r = sum(counts)
    off = offsets_of(counts)
    x, w, dy = normal(g, r, k, dtype=BF16), normal(g, len(counts), n, k, scale=k**-0.5, dtype=BF16), normal(g, r, n, dtype=BF16)
    check_mm(ex, x, w, off)
    check_mm(ex, dy, w.transpose(1, 2), off)
    check_wgrad(ex, dy, x, off)


def test_grouped_mm_strides_and_alignment(ex):
    g = gen(21)
    counts = [40, 0, 77, 130]
    r, n, k = sum(counts), 96, 128
    off = offsets_of(counts)
    wide = normal(g, r, 400, dtype=BF16)
    weights = normal(g, 4, 200, 300, scale=0.1, dtype=BF16)
    for shift in (0, 1, 4, 8):  # of the first column: alignments of 16, 2, 8 and 16 bytes
        x = wide[:, shift:shift + k]
        for w in (weights[:, :n, shift:shift + k], weights[:, shift:shift + k, :n].transpose(1, 2),
                  weights[:, 3:3 + n, :k].contiguous(), weights[:1, :n, :k].expand(4, n, k)):
            check_mm(ex, x, w, off)
        check_wgrad(ex, wide[:, shift + k:shift + k + n], x, off)
    # neither dimension of the weights is contiguous, rows of x overlap: copied, not refused
    assert torch.equal(ex.grouped_mm(wide[:, :k], weights[:, :2 * n:2, :2 * k:2], off),
                       ex.grouped_mm(wide[:, :k], weights[:, :2 * n:2, :2 * k:2].contiguous(), off))
    assert torch.equal(ex.grouped_mm(wide[:1, :k].expand(r, k), weights[:, :n, :k], off),
                       ex.grouped_mm(wide[:1, :k].repeat(r, 1), weights[:, :n, :k], off))


@pytest.mark.parametrize("r", [1, 2, 40])
@pytest.mark.parametrize("n,k,strides", [(64, 72, (64 * 72 + 1, 72, 1)), (64, 72, (0, 72, 1)), (1, 64, (3, 5, 1)), (64, 1, (7, 1, 3)),
                                         (1, 1, (2, 3, 5)), (72, 64, (5, 1, 72))])
def test_grouped_mm_strides_of_single_experts_and_features(ex, r, n, k, strides):
    """A dimension of size 1 may have any stride."""
    g = gen(22)
    w = normal(g, 8000, dtype=BF16).as_strided((1, n, k), strides)
    x = normal(g, r, k, dtype=BF16)
    off = offsets_of([r])
    check_mm(ex, x, w, off)
    check_mm(ex, normal(g, r, n, dtype=BF16), w.transpose(1, 2), off)
    leaf = w.detach().requires_grad_(True)
    (dw,) = torch.autograd.grad(ex.grouped_mm(x, leaf, off).sum(), leaf)
    size = x.double().abs().sum(0)
    assert ((dw.double() - x.double().sum(0)).abs() <= ULP[BF16] * x.double().sum(0).abs() + ACC * size * min(r, 64)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n,k", [(64, 128), (256, 256), (200, 320)])
def test_grouped_mm_keeps_groups_apart(ex, bad, n, k):
    """Infinities and NaN in the rows of one expert, or of none, reach no other expert's results."""
    g = gen(31)
    counts = [37, 20, 140, 1, 70]
    r = sum(counts) + 30
    off = offsets_of(counts)
    x, w, dy = normal(g, r, k, dtype=BF16), normal(g, 5, n, k, scale=0.1, dtype=BF16), normal(g, r, n, dtype=BF16)
    clean = ex._mm(x, None, r, w, off), ex._mm(dy, None, r, w, off, transposed=True), ex._wgrad(dy, x, off)
    x2, dy2 = x.clone(), dy.clone()
    lo, hi = 37, 57
    for t in (x2, dy2):
        t[lo:hi] = bad
        t[sum(counts):] = bad
    w2 = w.clone()
    w2[1] = bad
    out, dx, dw = ex._mm(x2, None, r, w2, off), ex._mm(dy2, None, r, w2, off, transposed=True), ex._wgrad(dy2, x2, off)
    keep = torch.ones(r, dtype=torch.bool, device="cuda")
    keep[lo:hi] = False
    assert torch.equal(out[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert not torch.isfinite(out[lo:hi]).any()
    others = [0, 2, 3, 4]
    assert torch.equal(dw[others], clean[2][others]) and not torch.isfinite(dw[1]).any()


def test_grouped_mm_offsets_outside_the_rows(ex):
    """Offsets past the rows, or that decrease, are taken as their running maximum within the rows."""
    g = gen(41)
    x, w = normal(g, 100, 64, dtype=BF16), normal(g, 4, 64, 64, scale=0.1, dtype=BF16)
    for odd, even in (([0, 40, 30, 1 << 30, 5], [0, 40, 40, 100, 100]), ([0, -5, 20, 20, 2147483647], [0, 0, 20, 20, 100])):
        a, b = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (odd, even))
        assert torch.equal(ex._mm(x, None, 100, w, a), ex._mm(x, None, 100, w, b))
        assert torch.equal(ex._wgrad(x, x, a), ex._wgrad(x, x, b))


def test_grouped_mm_row_numbers_outside_the_tokens(ex):
    g = gen(42)
    x, w = normal(g, 50, 64, dtype=BF16), normal(g, 2, 96, 64, scale=0.1, dtype=BF16)
    rows = torch.randint(0, 50, (300,), generator=g, device="cuda", dtype=torch.int32)
    rows[7], rows[150], rows[299] = -3, 50, 2147483647
    off = offsets_of([160, 140])
    out = ex._mm(x, rows, 300, w, off)
    assert (out[[7, 150, 299]] == 0).all()
    zeros = torch.cat([x, x.new_zeros(1, 64)])
    good = torch.where((rows >= 0) & (rows < 50), rows, 50).to(torch.int32)
    assert torch.equal(out, ex._mm(zeros, good, 300, w, off))
    assert torch.equal(ex._gather(x, rows), zeros[good.long()])


def test_grouped_mm_weights_past_32_bits(ex):
    """Element offsets of the last expert's weights, and of its gradient, do not fit 32 bits."""
    e, n, k = 140, 4096, 4096
    g = gen(43)
    w = torch.empty(e, n, k, dtype=BF16, device="cuda")
    w[-1] = normal(g, n, k, scale=k**-0.5)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    for r in (2, 40, 300):
        off[-1] = r
        x = normal(g, r, k, dtype=BF16)
        want, size = x.double() @ w[-1].double().T, x.double().abs() @ w[-1].double().abs().T
        within(ex._mm(x, None, r, w, off), want, ULP[BF16] * want.abs() + ACC * 64 * size)
        dw = ex._wgrad(x, x, off)
        assert not dw[:-1].any()
        want, size = x.double().T @ x.double(), x.double().abs().T @ x.double().abs()
        within(dw[-1], want, ULP[BF16] * want.abs() + ACC * 64 * size)


def test_grouped_mm_gradients_against_differences(ex):
    """The product is linear in either argument: a difference of any length gives the directional derivative."""
    g = gen(44)
    routing = ex.route_tokens(normal(g, 90, 6), 2)
    x, w = normal(g, 90, 160, dtype=FP16).requires_grad_(True), normal(g, 6, 80, 160, scale=0.1, dtype=FP16).requires_grad_(True)
    dy = normal(g, 180, 80, dtype=FP16)
    y = ex.grouped_mm(x, w, routing, gather=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ex_x, ex_w = normal(g, 90, 160, dtype=FP16), normal(g, 6, 80, 160, scale=0.1, dtype=FP16)
    with torch.no_grad():
        for grad, d, other in ((dx, ex_x, ex.grouped_mm(ex_x, w, routing, gather=True)),
                               (dw, ex_w, ex.grouped_mm(x, ex_w, routing, gather=True))):
            a, b = (grad.double() * d.double()).sum(), (dy.double() * other.double()).sum()
            size = (dy.double().abs() * other.double().abs()).sum() + (grad.double().abs() * d.double().abs()).sum()
            assert (a - b).abs() <= 3 * ULP[FP16] * size


# ---------------------------------------------------------------------------------------------------------------
# Gated activation
# ---------------------------------------------------------------------------------------------------------------


def held_in_8_bits(v):
    """The checkpoint's values in 64 bits, block by block; NaN throughout a block with an infinity or a NaN."""
    out = v.double().clone()
    for c in range(0, v.shape[1], 32):
        b = v[:, c:c + 32].double()
        top = b.abs().amax(1, keepdim=True)
        fine = torch.isfinite(b).all(1, keepdim=True)
        top = torch.where(fine, top, 1.0)
        e = torch.floor(torch.log2(top.clamp_min(2.0**-126))) - 6
        e = torch.where(torch.round(top * torch.exp2(-e)) > 127, e + 1, e).clamp_min(-126)
        out[:, c:c + 32] = torch.where(fine, torch.round(b * torch.exp2(-e)) * torch.exp2(e), math.nan)
    return out


def routing_of(ex, r, gates, pairs):
    position = torch.full((r,), -1, dtype=torch.int32, device="cuda")
    live = pairs >= 0
    position[pairs[live].long()] = torch.arange(r, dtype=torch.int32, device="cuda")[live]
    zeros = torch.zeros(r, 1, dtype=torch.int32, device="cuda")
    return ex.Routing(gates, zeros, torch.tensor([0, int(live.sum())], dtype=torch.int32, device="cuda"), pairs, pairs.clone(),
                      position.reshape(r, 1))


def some_routing(ex, g, r, off):
    pairs = torch.randperm(r, generator=g, device="cuda").to(torch.int32)
    if off:
        pairs[-off:] = -1
    return routing_of(ex, r, torch.rand(r, 1, generator=g, device="cuda"), pairs)


def act_reference(u, p, dh, checkpoint):
    f = u.shape[1] // 2
    g, v = u[:, :f].double(), u[:, f:].double()
    h = p * (g * torch.sigmoid(g)) * v
    if checkpoint:
        g, v = held_in_8_bits(u[:, :f]), held_in_8_bits(u[:, f:])
    s, d = torch.sigmoid(g), dh.double()
    dg, dv = p * d * v * (s + g * s * (1 - s)), p * d * g * s
    size = torch.cat([(p * d * v).abs() * (s + (g * s).abs()), (p * d * g * s).abs()], 1)
    return h, torch.cat([dg, dv], 1), size, d * g * s * v


@pytest.mark.parametrize("r,f", [(1, 1), (3, 31), (5, 32), (2, 33), (17, 100), (4, 256), (9, 264), (6, 1100), (300, 2048), (3000, 64),
                                 (1, 4100)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("checkpoint", [True, False])
def test_gated_act(ex, r, f, dtype, checkpoint):
    g = gen(r * 31 + f)
    u, dh = normal(g, r, 2 * f, scale=2.0, dtype=dtype), normal(g, r, f, dtype=dtype)
    for routing in (None, some_routing(ex, g, r, r // 4)):
        ul = u.clone().requires_grad_(True)
        if routing is None:
            p = torch.ones(r, 1, dtype=torch.float64, device="cuda")
        else:
            routing = routing._replace(gates=routing.gates.requires_grad_(True))
            live = routing.pairs >= 0
            p = (routing.gates.detach().double()[routing.pairs.long().clamp_min(0), 0] * live)[:, None]
        h = ex.gated_act(ul, routing, checkpoint=checkpoint)
        want, du, size, per = act_reference(u, p, dh, checkpoint)
        within(h, want, (ULP[dtype] + FUN) * want.abs() + TINY[dtype])
        leaves = (ul,) if routing is None else (ul, routing.gates)
        got = torch.autograd.grad(h, leaves, dh)
        within(got[0], du, ULP[dtype] * du.abs() + FUN * size + TINY[dtype])
        if routing is not None:
            dp = torch.zeros(r, dtype=torch.float64, device="cuda")
            dp[routing.pairs[live].long()] = per.sum(1)[live]
            mag = torch.zeros(r, dtype=torch.float64, device="cuda")
            mag[routing.pairs[live].long()] = per.abs().sum(1)[live]
            within(got[1][:, 0], dp, (FUN + f * 2.0**-24) * mag + 1e-37)
        with torch.no_grad():
            assert torch.equal(ex.gated_act(u, routing), h)


def test_gated_act_extreme_blocks(ex):
    """Zeros, the type's smallest and largest values, a block with an infinity or a NaN beside a good one, 127.5 steps."""
    f = 96
    u = torch.ones(8, 2 * f, device="cuda")
    u[0] = 0
    u[1, :32], u[1, 32:64] = 1e-40, 2.0**-126
    u[2, :32] = torch.linspace(-127.4999, 127.4999, 32, device="cuda")
    u[3, :32] = torch.linspace(-127.5, 127.5, 32, device="cuda")
    u[4, 5] = math.inf
    u[5, f + 40] = math.nan
    u[6, :] = 3.0e38
    u[7, f:] = torch.arange(f, device="cuda") * 0.5
    h, held = ex._act(u, None, None, True)
    codes, scales = held[:8 * 2 * f].view(torch.int8).view(8, 2 * f), held[8 * 2 * f:].view(8, 6)
    for half in range(2):
        v = u[:, half * f:(half + 1) * f]
        got = codes[:, half * f:(half + 1) * f].double() * torch.exp2(scales[:, 3 * half:3 * half + 3].double() - 127).repeat_interleave(32, 1)
        want = held_in_8_bits(v)
        bad = torch.isnan(want)
        assert torch.equal(scales[:, 3 * half:3 * half + 3].repeat_interleave(32, 1) == 255, bad)
        assert torch.equal(got[~bad], want[~bad])
        err = (got - v.double()).abs()[~bad]
        top = v.double().reshape(8, 3, 32).abs().amax(2).repeat_interleave(32, 1)[~bad]
        assert (err <= top / 128 + 2.0**-127).all()
    du, _, _ = ex._act_grad(None, held, None, None, None, torch.ones(8, f, device="cuda"), False, False)
    assert torch.isnan(du[4, :32]).all() and torch.isfinite(du[4, 32:f]).all() and torch.isfinite(du[[0, 1, 2, 3, 7]]).all()


def test_gated_act_rows_of_no_pair_do_not_show(ex):
    g = gen(52)
    u = normal(g, 20, 128, dtype=BF16)
    u[10:] = math.nan
    pairs = torch.cat([torch.arange(10), torch.full((10,), -1)]).to(dtype=torch.int32, device="cuda")
    routing = routing_of(ex, 20, torch.rand(20, 1, generator=g, device="cuda").requires_grad_(True), pairs)
    ul = u.clone().requires_grad_(True)
    h = ex.gated_act(ul, routing)
    du, dp = torch.autograd.grad(h, (ul, routing.gates), torch.full_like(h, math.nan).index_fill(0, torch.arange(10, device="cuda"), 1.0))
    assert (h[10:] == 0).all() and (du[10:] == 0).all() and (dp[10:] == 0).all() and torch.isfinite(du).all() and torch.isfinite(h).all()


def test_gated_act_gradient_against_differences(ex):
    g = gen(53)
    u, d, w = normal(g, 30, 80), normal(g, 30, 80), normal(g, 30, 40)
    for checkpoint in (True, False):
        ul = u.clone().requires_grad_(True)
        (du,) = torch.autograd.grad(ex.gated_act(ul, checkpoint=checkpoint), (ul,), w)
        at = torch.cat([held_in_8_bits(u[:, :40]), held_in_8_bits(u[:, 40:])], 1) if checkpoint else u.double()
        h = 1e-5
        f = lambda z: (torch.nn.functional.silu(z[:, :40]) * z[:, 40:] * w.double()).sum(1)
        diff = (f(at + h * d.double()) - f(at - h * d.double())) / (2 * h)
        size = (du.abs() * d.abs()).sum(1).double() + 1
        assert ((du.double() * d.double()).sum(1) - diff).abs().le(1e-5 * size).all()


def test_gated_act_strides(ex):
    g = gen(54)
    wide = normal(g, 60, 700, dtype=BF16)
    for shift in (0, 1, 4):
        u = wide[:, shift:shift + 512]
        ul = u.detach().requires_grad_(True)
        h = ex.gated_act(ul)
        assert torch.equal(h, ex.gated_act(u.contiguous()))
        dh = wide[:, shift + 100:shift + 356]
        u2 = u.contiguous().requires_grad_(True)
        a, = torch.autograd.grad(h, (ul,), dh)
        b, = torch.autograd.grad(ex.gated_act(u2), (u2,), dh.contiguous())
        assert torch.equal(a, b)


def test_gated_act_past_32_bits(ex):
    r, f = 300_000, 4096
    g = gen(55)
    u = torch.zeros(r, 2 * f, dtype=BF16, device="cuda")
    u[-3:] = normal(g, 3, 2 * f)
    ul = u.requires_grad_(True)
    h = ex.gated_act(ul)
    dh = torch.ones_like(h)
    (du,) = torch.autograd.grad(h, (ul,), dh)
    want, dwant, size, _ = act_reference(u.detach()[-3:], 1.0, dh[-3:], True)
    within(h[-3:], want, (ULP[BF16] + FUN) * want.abs())
    within(du[-3:], dwant, ULP[BF16] * dwant.abs() + FUN * size)
    assert not h[:-3].any() and not du[:-3].any()


# ---------------------------------------------------------------------------------------------------------------
# Back into tokens
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t,k,d", [(1, 1, 1), (1, 4, 2048), (7, 3, 33), (37, 4, 1100), (300, 2, 300), (513, 8, 264), (40, 32, 72)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(ex, t, k, d, dtype, weighted):
    g = gen(t + k + d)
    logits = normal(g, t, 40)
    routing = ex.route_tokens(logits, k, mask=torch.arange(t, device="cuda") % 5 != 2)
    routing = routing._replace(gates=routing.gates.clone().requires_grad_(True))
    o = normal(g, t * k, d, dtype=dtype)
    o[int(routing.offsets[-1]):] = math.nan  # rows of no pair
    ol, dy = o.clone().requires_grad_(True), normal(g, t, d, dtype=dtype)
    y = ex.combine_rows(ol, routing, weighted=weighted)
    pos, live = routing.position.long().clamp_min(0), routing.position >= 0
    w = (routing.gates.detach().double() if weighted else torch.ones(t, k, dtype=torch.float64, device="cuda")) * live
    terms = torch.where(live[..., None], w[..., None] * o.double()[pos], 0.0)
    within(y, terms.sum(1), ULP[dtype] * terms.sum(1).abs() + k * 2.0**-23 * terms.abs().sum(1) + TINY[dtype])
    got = torch.autograd.grad(y, (ol, routing.gates) if weighted else (ol,), dy)
    do = torch.zeros(t * k, d, dtype=torch.float64, device="cuda")
    do[pos[live]] = (w[..., None] * dy.double()[:, None, :])[live]
    within(got[0], do, (ULP[dtype] + 2.0**-24) * do.abs() + TINY[dtype])
    if weighted:
        per = torch.where(live[..., None], o.double()[pos] * dy.double()[:, None, :], 0.0)
        within(got[1], per.sum(2), d * 2.0**-24 * per.abs().sum(2) + 1e-37)


def test_combine_strides_and_positions_outside(ex):
    g = gen(61)
    routing = ex.route_tokens(normal(g, 50, 9), 2)
    wide = normal(g, 100, 500, dtype=BF16)
    for shift in (0, 1, 4):
        assert torch.equal(ex.combine_rows(wide[:, shift:shift + 256], routing),
                           ex.combine_rows(wide[:, shift:shift + 256].contiguous(), routing))
    position = routing.position.clone()
    position[3, 0], position[4, 1] = 100, -7
    gates = routing.gates.clone()
    gates[3, 0] = gates[4, 1] = 0
    o = wide[:, :64].contiguous()
    assert torch.equal(ex.combine_rows(o, routing._replace(position=position)), ex.combine_rows(o, routing._replace(gates=gates)))


def test_combine_gradients_against_differences(ex):
    """The sum is linear in the rows and in the gates: a difference of any length gives the directional derivative."""
    g = gen(62)
    routing = ex.route_tokens(normal(g, 70, 9), 3, mask=torch.arange(70, device="cuda") % 8 != 1)
    gates = routing.gates.clone().requires_grad_(True)
    o, dy = normal(g, 210, 130).requires_grad_(True), normal(g, 70, 130)
    do, dg = torch.autograd.grad(ex.combine_rows(o, routing._replace(gates=gates)), (o, gates), dy)
    eo, eg = normal(g, 210, 130), normal(g, 70, 3) * (routing.position >= 0)
    with torch.no_grad():
        for grad, step, moved in ((do, eo, ex.combine_rows(eo, routing)), (dg, eg, ex.combine_rows(o, routing._replace(gates=eg)))):
            a, b = (grad.double() * step.double()).sum(), (dy.double() * moved.double()).sum()
            size = (grad.double() * step.double()).abs().sum() + (dy.double() * moved.double()).abs().sum()
            assert (a - b).abs() <= 2.0**-20 * size


# ---------------------------------------------------------------------------------------------------------------
# The layer, and how all of it behaves as a part of a program
# ---------------------------------------------------------------------------------------------------------------


def layer(ex, g, t, d, f, e, k, dtype=BF16):
    x = normal(g, t, d, dtype=dtype)
    w_in, w_out = normal(g, e, 2 * f, d, scale=d**-0.5, dtype=dtype), normal(g, e, d, f, scale=f**-0.5, dtype=dtype)
    return x, w_in, w_out, normal(g, t, e)


def plain_layer(x, w_in, w_out, gates, experts):
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    f = w_out.shape[2]
    for e in range(w_in.shape[0]):
        token, slot = (experts == e).nonzero(as_tuple=True)
        if len(token):
            u = x[token] @ w_in[e].T
            h = torch.nn.functional.silu(u[:, :f]) * u[:, f:] * gates[token, slot][:, None]
            y = y.index_add(0, token, h @ w_out[e].T)
    return y


@pytest.mark.parametrize("t,d,f,e,k", [(1, 128, 64, 4, 2), (70, 256, 192, 8, 3), (400, 136, 100, 5, 2)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("checkpoint", [True, False])
def test_expert_mlp(ex, t, d, f, e, k, dtype, checkpoint):
    g = gen(t + d)
    x, w_in, w_out, logits = layer(ex, g, t, d, f, e, k, dtype)
    leaves = [v.requires_grad_(True) for v in (x, w_in, w_out, logits)]
    routing = ex.route_tokens(logits, k, mask=torch.arange(t, device="cuda") % 6 != 5)
    y = ex.expert_mlp(x, w_in, w_out, routing, checkpoint=checkpoint)
    dy = normal(g, t, d, dtype=dtype)
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)

    dl = [v.detach().double().requires_grad_(True) for v in leaves]
    chosen, live = routing.experts.long().clamp_min(0), routing.experts >= 0
    gates = torch.softmax(dl[3].gather(1, chosen), 1) * live
    want = plain_layer(dl[0], dl[1], dl[2], gates, routing.experts)
    wants = torch.autograd.grad(want, dl, dy.double())
    # each of the chain's tensors is rounded once: u, h, the rows of the second product, the sum; the gradients also pass
    # dh, du and the rows of dx, and with the checkpoint u in steps of 1/128 of a block's maximum (about 1/60 of a
    # standard deviation, half of it at most, to first order in each of two factors)
    norm = lambda a, b: ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()
    assert norm(y, want) < 4 * 2 * ULP[dtype]
    for a, b in zip(got, wants):
        assert norm(a, b) < 8 * 2 * ULP[dtype] + (0.02 if checkpoint else 0.0)
    with torch.no_grad():
        assert torch.equal(ex.expert_mlp(x, w_in, w_out, routing), y)
    # the layer is its parts
    u = ex.grouped_mm(x, w_in, routing, gather=True)
    h = ex.gated_act(u, routing, checkpoint=checkpoint)
    y2 = ex.combine_rows(ex.grouped_mm(h, w_out, routing), routing, weighted=False)
    assert torch.equal(y, y2)
    dx, dlog = torch.autograd.grad(y2, (x, logits), dy)
    assert norm(dx, got[0].double()) < 8 * 2 * ULP[dtype] and norm(dlog, got[3].double()) < 8 * 2 * ULP[dtype]


def test_expert_mlp_gradient_against_differences(ex):
    """Differences of the layer in 64 bits along one direction of all its inputs, against the fp16 layer's gradients."""
    g = gen(70)
    t, d, f, e, k = 120, 96, 80, 6, 2
    x, w_in, w_out, logits = layer(ex, g, t, d, f, e, k, FP16)
    leaves = [v.requires_grad_(True) for v in (x, w_in, w_out, logits)]
    routing = ex.route_tokens(logits, k)
    dy = normal(g, t, d, dtype=FP16)
    grads = torch.autograd.grad(ex.expert_mlp(x, w_in, w_out, routing, checkpoint=False), leaves, dy)
    steps = [normal(g, *v.shape).double() * v.detach().double().std() for v in leaves]
    chosen = routing.experts.long()

    def value(h):
        a, b, c, l = (v.detach().double() + h * s for v, s in zip(leaves, steps))
        return (plain_layer(a, b, c, torch.softmax(l.gather(1, chosen), 1), routing.experts) * dy.double()).sum()

    diff = (value(1e-4) - value(-1e-4)) / 2e-4
    got = sum((a.double() * s).sum() for a, s in zip(grads, steps))
    # six tensors rounded to fp16 between input and gradient, none of them along the direction in particular; the sums of
    # thousands of such terms are compared by their magnitudes' root sum of squares
    size = math.sqrt(sum(((a.double() * s) ** 2).sum().item() for a, s in zip(grads, steps)))
    assert (got - diff).abs().item() <= 40 * 6 * ULP[FP16] * size


def test_same_bits_in_every_run_and_on_another_stream(ex):
    g = gen(71)
    x, w_in, w_out, logits = layer(ex, g, 900, 256, 320, 12, 4)
    leaves = [v.requires_grad_(True) for v in (x, w_in, w_out, logits)]

    def step():
        y = ex.expert_mlp(x, w_in, w_out, ex.route_tokens(logits, 4))
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        others = [step() for _ in range(3)]
    side.synchronize()
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_forward_in_a_cuda_graph_follows_its_inputs(ex):
    g = gen(72)
    x, w_in, w_out, logits = layer(ex, g, 48, 256, 128, 16, 2)
    step = lambda: ex.expert_mlp(x, w_in, w_out, ex.route_tokens(logits, 2))
    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        for seed in (1, 2):
            x.copy_(normal(gen(seed), 48, 256))
            logits.copy_(normal(gen(seed + 9), 48, 16))  # other groups, other sizes
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, step())


def test_empty_batches(ex):
    x, w_in, w_out, logits = layer(ex, gen(73), 0, 64, 32, 4, 2)
    leaves = [v.requires_grad_(True) for v in (x, w_in, w_out, logits)]
    routing = ex.route_tokens(logits, 2)
    y = ex.expert_mlp(x, w_in, w_out, routing)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert y.shape == (0, 64) and routing.offsets.tolist() == [0] * 5
    assert not grads[1].any() and not grads[2].any() and grads[0].shape == (0, 64)


def test_transport_bias_evens_the_loads(ex):
    g = gen(74)
    t, d, e = 4096, 64, 16
    x = normal(g, t, d) + normal(g, 1, d)  # a common direction: some experts are far more popular
    router = normal(g, e, d, scale=d**-0.5)
    logits = x @ router.t()
    before = ex.route_tokens(logits, 1).offsets.diff().float()
    bias = ex.transport_bias(x, router, eps=0.05, n_iters=200, allow_tf32=False)
    after = ex.route_tokens(logits, 1, bias=bias).offsets.diff().float()
    assert before.max() > 2 * t / e and after.max() < 1.25 * t / e and after.min() > 0.75 * t / e
    # marginals of the plan that the prices belong to
    plan = torch.softmax((logits.double() + bias.double()) / 0.05, 1)
    assert (plan.mean(0) * e - 1).abs().max() < 0.05


def test_refusals(ex):
    g = gen(75)
    cpu = torch.zeros(4, 8)
    x, w_in, w_out, logits = layer(ex, g, 6, 64, 32, 4, 2)
    r = ex.route_tokens(logits, 2)
    off = r.offsets
    bad = [
        lambda: ex.route_tokens(cpu, 2), lambda: ex.route_tokens(logits[0], 2), lambda: ex.route_tokens(logits, 0),
        lambda: ex.route_tokens(logits, 5), lambda: ex.route_tokens(logits.double(), 2),
        lambda: ex.route_tokens(torch.zeros(2, 1025, device="cuda"), 2),
        lambda: ex.route_tokens(torch.zeros(2, 64, device="cuda"), 33),
        lambda: ex.route_tokens(logits, 2, bias=torch.zeros(3, device="cuda")),
        lambda: ex.route_tokens(logits, 2, bias=torch.zeros(4, device="cuda", requires_grad=True)),
        lambda: ex.route_tokens(logits, 2, mask=torch.ones(6, device="cuda")),
        lambda: ex.route_tokens(logits, 2, normalize="none"),
        lambda: ex.grouped_mm(x.float(), w_in.float(), r, gather=True), lambda: ex.grouped_mm(x, w_in.half(), r, gather=True),
        lambda: ex.grouped_mm(x, w_in, r), lambda: ex.grouped_mm(x, w_in, off.long()), lambda: ex.grouped_mm(x, w_in, off, gather=True),
        lambda: ex.grouped_mm(x, w_in[:3], r, gather=True), lambda: ex.grouped_mm(x[:, :32], w_in, r, gather=True),
        lambda: ex.grouped_mm(x[0], w_in, r), lambda: ex.grouped_mm(x, w_in, off.cpu()),
        lambda: ex.grouped_mm(x, w_in, r._replace(rows=r.rows[:-1]), gather=True),
        lambda: ex.gated_act(cpu), lambda: ex.gated_act(x[:, :7]), lambda: ex.gated_act(x, r), lambda: ex.gated_act(x.double()),
        lambda: ex.gated_act(x, tuple(r)), lambda: ex.combine_rows(x, r), lambda: ex.combine_rows(x[0], r),
        lambda: ex.combine_rows(x.double(), r), lambda: ex.combine_rows(cpu, r),
        lambda: ex.expert_mlp(x, w_in, w_out.half(), r), lambda: ex.expert_mlp(x[:5], w_in, w_out, r),
        lambda: ex.expert_mlp(x, w_in[:, :-2], w_out, r), lambda: ex.expert_mlp(x.float(), w_in.float(), w_out.float(), r),
        lambda: ex.route_tokens(logits, 2, bias=torch.zeros(4)), lambda: ex.grouped_mm(x, w_in.cpu(), r, gather=True),
        lambda: ex.transport_bias(x, logits), lambda: ex.transport_bias(x[:0], w_in[0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_gradients_are_not_differentiable_again(ex):
    g = gen(76)
    x, w_in, w_out, logits = layer(ex, g, 6, 64, 32, 4, 2)
    x.requires_grad_(True)
    y = ex.expert_mlp(x, w_in, w_out, ex.route_tokens(logits, 2))
    (dx,) = torch.autograd.grad(y, (x,), torch.ones_like(y), create_graph=True)
    assert torch.isfinite(dx).all()
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dx.float().sum().backward()


def test_a_failed_call_raises_the_library_s_error(ex):
    from flash_sinkhorn_b200 import _lib
    x, w = torch.zeros(4, 8, dtype=BF16, device="cuda"), torch.zeros(2000, 8, 8, dtype=BF16, device="cuda")
    with pytest.raises(_lib.FlashSinkhornError, match="FS_ERR_BAD_ARG"):
        ex._mm(x, None, 4, w, torch.zeros(2001, dtype=torch.int32, device="cuda"))
