"""Routed experts at the ends of their ranges: magnitudes, sizes, threads, derivatives that are not theirs to give.

Bounds are those of the operators' other tests: half a unit in the last place for each rounding to the type, ``FUN`` for
the sigmoid and the products around it, ``ACC`` per term of a sum in fp32.
"""
import os
import subprocess
import sys
import threading

import pytest
import torch

from test_gpu_experts import (ACC, BF16, FP16, FP32, FUN, TINY, ULP, act_reference, check_mm, check_wgrad, ex, gen, held_in_8_bits, normal,  # noqa: F401
                              offsets_of, within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def no_wait_gave_up():
    from flash_sinkhorn_b200 import _lib
    yield
    assert _lib.load().fs_device_error() == 0


def large_blocks(dtype, top, seed):
    """Rows [g | v] of one block each: a large g beside an ordinary v, and the other way round; zeros and ones in the large one."""
    g = gen(seed)
    rows = []
    for big_first in (True, False):
        for power in (104, 105, 110, 111, 112, 119, 120, 126, 127):
            big = (torch.rand(32, generator=g, device="cuda") * 2 - 1) * (top * 2.0**power)
            big[0], big[1], big[2], big[3] = top * 2.0**power, -top * 2.0**power, 0.0, 1.0
            small = torch.rand(32, generator=g, device="cuda") * 0.9 - 0.45
            rows.append(torch.cat([big, small] if big_first else [small, big]))
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gated_act_checkpoint_of_large_values(ex, dtype):  # noqa: F811
    """Blocks up to the end of the type's range come back as their codes say, and their gradients with them."""
    u = large_blocks(dtype, 1.984375, 1)  # 127 / 64: the largest of a block is its 127th step
    dh = normal(gen(2), u.shape[0], 32, scale=2.0**-40, dtype=dtype)
    h, held = ex._act(u, None, None, True)
    du, _, again = ex._act_grad(None, held, None, None, None, dh, False, True)
    want, dwant, size, _ = act_reference(u, 1.0, dh, True)
    within(h, want, (ULP[dtype] + FUN) * want.abs() + TINY[dtype])
    within(du, dwant, ULP[dtype] * dwant.abs() + FUN * size + TINY[dtype])
    held_u = torch.cat([held_in_8_bits(u[:, :32]), held_in_8_bits(u[:, 32:])], 1)
    want = act_reference(held_u, 1.0, dh, False)[0]
    within(again, want, (ULP[dtype] + FUN) * want.abs() + TINY[dtype])
    leaf = u.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ex.gated_act(leaf), leaf, dh)[0], du)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gated_act_checkpoint_of_the_largest_values(ex, dtype):  # noqa: F811
    """A largest magnitude that rounds up to 2^128 stands for the largest of fp32: within 1/128 of itself, not an infinity."""
    top = torch.finfo(dtype).max
    u = torch.ones(4, 64, device="cuda", dtype=dtype)
    u[0, 0], u[1, 0], u[2, 32], u[3, 40] = top, -top, top, -top
    u[:2, 1], u[2:, 33] = 0.5 * top, -0.25 * top  # 32 and 16 steps of 2^122
    u[:2, 32:] *= 0.25
    dh = torch.full((4, 32), 2.0**-40, device="cuda", dtype=dtype)
    h, held = ex._act(u, None, None, True)
    du, _, again = ex._act_grad(None, held, None, None, None, dh, False, True)
    held_u = torch.cat([held_in_8_bits(u[:, :32]), held_in_8_bits(u[:, 32:])], 1).clamp(-torch.finfo(FP32).max, torch.finfo(FP32).max)
    assert ((held_u - u.double()).abs() <= u.double().abs().reshape(4, 2, 32).amax(2).repeat_interleave(32, 1) / 128).all()
    want, dwant, size, _ = act_reference(held_u, 1.0, dh, False)
    within(du, dwant, ULP[dtype] * dwant.abs() + FUN * size + TINY[dtype])
    fits = want.abs() < top * (1 - 2 * ULP[dtype])  # 0.73 and 0.25 times the largest
    within(again[fits], want[fits], (ULP[dtype] + FUN) * want[fits].abs() + TINY[dtype])
    assert fits.all() and torch.isfinite(h).all()


def test_routing_from_several_threads(ex):  # noqa: F811
    """Threads whose routings need different amounts of shared memory do not take it from one another."""
    failed, outputs = [], {}

    def work(name, e, k, tokens, times):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                logits = normal(gen(e), tokens, e).requires_grad_(True)
                for i in range(times):
                    r = ex.route_tokens(logits, k, normalize="all")
                    (d,) = torch.autograd.grad(r.gates, (logits,), torch.ones_like(r.gates))
                    if i in (0, times - 1):
                        outputs[name, i > 0] = [v.detach().clone() for v in (*r, d)]
            torch.cuda.synchronize()
        except Exception as error:
            failed.append((name, str(error)))

    sizes = [(1024, 2, 500), (512, 2, 500), (400, 3, 300), (1024, 4, 40), (700, 1, 64), (370, 2, 200)]
    threads = [threading.Thread(target=work, args=(i, *size, 1000)) for i, size in enumerate(sizes)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed[:3]
    for i in range(len(sizes)):
        assert all(torch.equal(a, b) for a, b in zip(outputs[i, False], outputs[i, True]))


@pytest.mark.parametrize("mode", ["gradients", "no_grad"])
def test_forward_mode_derivatives_are_refused(ex, mode):  # noqa: F811
    """A tangent is not dropped, which would count as a derivative of zero."""
    g = gen(5)
    logits, u, o, gates = normal(g, 6, 8), normal(g, 12, 64), normal(g, 12, 32), torch.rand(6, 2, device="cuda")
    x, w, w_in, w_out = (normal(g, *s, dtype=BF16) for s in ((12, 64), (8, 16, 64), (8, 32, 32), (8, 32, 16)))
    y = normal(g, 6, 32, dtype=BF16)
    r = ex.route_tokens(logits, 2)
    off = r.offsets
    calls = [
        (lambda t: ex.route_tokens(t, 2), logits), (lambda t: ex.grouped_mm(t, w, off), x), (lambda t: ex.grouped_mm(x, t, off), w),
        (lambda t: ex.gated_act(t), u), (lambda t: ex.gated_act(u, r._replace(gates=t), checkpoint=False), gates),
        (lambda t: ex.combine_rows(t, r, weighted=False), o), (lambda t: ex.combine_rows(o, r._replace(gates=t)), gates),
        (lambda t: ex.expert_mlp(t, w_in, w_out, r), y), (lambda t: ex.expert_mlp(y, t, w_out, r), w_in),
        (lambda t: ex.expert_mlp(y, w_in, t, r), w_out), (lambda t: ex.expert_mlp(y, w_in, w_out, r._replace(gates=t)), gates),
    ]
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(mode == "gradients"):
        for i, (call, t) in enumerate(calls):
            with pytest.raises(RuntimeError, match="jvp"):
                call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
                pytest.fail(f"call {i} was not refused")
    for call, t in calls:  # without a tangent they go through
        call(t)


# copied: tiles of 128 rows and 128 features are more than 148 (6,000 rows: 147), and there are more than 256 features
@pytest.mark.parametrize("tokens,slots,e,n,k,copied", [(3000, 2, 4, 320, 200, 0), (4000, 2, 4, 320, 200, 1), (3000, 2, 4, 256, 200, 0),
                                                       (16384, 4, 64, 512, 256, 1), (16384, 4, 64, 256, 256, 0)])
def test_gathered_rows_go_to_single_ctas_or_are_copied(ex, tokens, slots, e, n, k, copied):  # noqa: F811
    """Rows in another order: products that want pairs of CTAs copy them first, and both ways give what the rows say."""
    from flash_sinkhorn_b200 import _lib
    lib, r = _lib.load(), tokens * slots
    assert lib.fs_grouped_mm_in_order(r, e, n) == copied
    g = gen(n + e)
    routing = ex.route_tokens(normal(g, tokens, e), slots, mask=torch.arange(tokens, device="cuda") % 7 != 3)
    x, w = normal(g, tokens, k, dtype=BF16), normal(g, e, n, k, scale=k**-0.5, dtype=BF16)
    by_binding = check_mm(ex, x, w, routing.offsets, routing.rows)
    out = torch.empty_like(by_binding)
    _lib.call("fs_grouped_mm", x.device, x.data_ptr(), k, tokens, routing.rows.data_ptr(), r, w.data_ptr(), n * k, k, 1, e, n, k,
              routing.offsets.data_ptr(), out.data_ptr(), 2, n, 2, _lib.stream_ptr(x.device))
    xs, ends, want = x.double()[routing.rows.long().clamp_min(0)], routing.offsets.tolist(), torch.zeros(r, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for j in range(e):
        want[ends[j]:ends[j + 1]] = xs[ends[j]:ends[j + 1]] @ w[j].double().T
        size[ends[j]:ends[j + 1]] = xs[ends[j]:ends[j + 1]].abs() @ w[j].double().abs().T
    within(out, want, ULP[BF16] * want.abs() + ACC * 64 * size + TINY[BF16])
    dy = normal(g, r, n, dtype=BF16)
    for _ in range(20):  # ends of groups in shared memory of both CTAs of a pair
        again = ex._wgrad(dy, ex._gather(x, routing.rows), routing.offsets)
    assert torch.equal(again, check_wgrad(ex, dy, ex._gather(x, routing.rows), routing.offsets))


@pytest.mark.parametrize("ctas,counts", [(0, [100_000_019]), (1, [99_999_984, 37])])
def test_weight_gradient_of_a_very_long_group(ex, ctas, counts):  # noqa: F811
    """One tile's products take longer than a single wait lasts (2^28 clocks): the warps behind them wait in proportion. In the
    second case the end that is zeroed comes a long tile after the warp that does so has started to wait."""
    from flash_sinkhorn_b200 import _lib
    lib, r = _lib.load(), sum(counts)
    g = gen(91)
    x = torch.zeros(r, 64, dtype=BF16, device="cuda")
    at = torch.cat([torch.randint(0, r, (100_000,), generator=g, device="cuda"), torch.arange(r - 60, r, device="cuda"),
                    torch.arange(60, device="cuda")]).unique()
    x[at] = torch.randint(-1, 2, (at.numel(), 64), generator=g, device="cuda").to(BF16)  # sums are exact in fp32 in any order
    want, ends = [], offsets_of(counts).tolist()
    for lo, hi in zip(ends[:-1], ends[1:]):
        rows = x[at[(at >= lo) & (at < hi)]].double()
        want.append((rows.T @ rows).to(BF16))
    before = lib.fs_set_cta_limit(ctas)
    try:
        got = ex._wgrad(x, x, offsets_of(counts))
        torch.cuda.synchronize()
    finally:
        lib.fs_set_cta_limit(before)
    assert lib.fs_device_error() == 0 and torch.equal(got, torch.stack(want))


# tiles of single CTAs (rows in order and one by one, weights of either layout), of pairs; sizes that end inside tiles
@pytest.mark.parametrize("tokens,e,n,k,gather", [(40, 3, 100, 72, False), (40, 3, 100, 72, True), (600, 3, 200, 328, False), (5000, 2, 700, 520, False),
                                                 (3000, 2, 1200, 1100, False), (9000, 2, 250, 136, True)])
def test_products_that_give_up(ex, tokens, e, n, k, gather):  # noqa: F811
    """Where a wait gives up, nothing passes for a result: NaN in what was not written, and the health word is set."""
    from flash_sinkhorn_b200 import _lib
    lib = _lib.load()
    g = gen(n)
    routing = ex.route_tokens(normal(g, tokens, e), 1, mask=torch.arange(tokens, device="cuda") % 8 != 5)
    off, routed = routing.offsets, int(routing.offsets[-1])
    x, w, dy = normal(g, tokens, k, dtype=BF16), normal(g, e, n, k, scale=k**-0.5, dtype=BF16), normal(g, tokens, n, dtype=BF16)
    rows = routing.rows if gather else None
    calls = [lambda: ex._mm(x, rows, tokens, w, off), lambda: ex._mm(dy, rows, tokens, w, off, transposed=True),
             lambda: ex._mm(dy, None, tokens, w, off, transposed=True, dtype=FP32), lambda: ex._wgrad(dy, x, off)]
    good = [call() for call in calls]
    for i, call in enumerate(calls):
        usual = lib.fs_set_product_limit(0)
        try:
            out = call()
            assert lib.fs_device_error() == 1
        finally:
            lib.fs_set_product_limit(usual)
            torch.cuda.synchronize()
            assert lib.fs_clear_device_error() == 0
        assert torch.isnan(out if i == 3 else out[:routed]).all() and (i == 3 or not out[routed:].any())
    assert lib.fs_device_error() == 0 and all(torch.equal(call(), want) for call, want in zip(calls, good))


@pytest.mark.parametrize("t,d,f,e,k", [(90, 136, 72, 6, 3), (257, 264, 128, 12, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_layer_sums_a_token_s_gradient_before_it_rounds(ex, t, d, f, e, k, dtype):  # noqa: F811
    """dx of the layer is that of its parts, element by element: the rows of a token are summed in fp32 and rounded once."""
    g = gen(t)
    x = normal(g, t, d, dtype=dtype).requires_grad_(True)
    w_in, w_out = normal(g, e, 2 * f, d, scale=d**-0.5, dtype=dtype), normal(g, e, d, f, scale=f**-0.5, dtype=dtype)
    routing, dy = ex.route_tokens(normal(g, t, e), k, mask=torch.arange(t, device="cuda") % 9 != 4), normal(g, t, d, dtype=dtype)
    (got,) = torch.autograd.grad(ex.expert_mlp(x, w_in, w_out, routing, checkpoint=False), x, dy)
    # the gradient of u as the layer has it, from the kernels by themselves; from there on in 64 bits
    r = t * k
    u = ex._mm(x.detach(), routing.rows, r, w_in, routing.offsets)
    dh = ex._mm(ex._gather(dy, routing.rows), None, r, w_out, routing.offsets, transposed=True)
    du = ex._act_grad(u, None, routing.gates, routing.pairs, routing.position, dh, False, False)[0].double()
    want, size = torch.zeros(t, d, dtype=torch.float64, device="cuda"), torch.zeros(t, d, dtype=torch.float64, device="cuda")
    ends = routing.offsets.tolist()
    for j, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        to = routing.rows[lo:hi].long()
        want.index_add_(0, to, du[lo:hi] @ w_in[j].double())
        size.index_add_(0, to, du[lo:hi].abs() @ w_in[j].double().abs())
    within(got, want, ULP[dtype] * want.abs() + ACC * 64 * size + TINY[dtype])


def nonzero_rows(t):
    """Rows of eight 16-bit values that hold anything but zeros of either sign."""
    words = t.view(torch.int64)
    return torch.cat([((words[c:c + (1 << 28), 0] | words[c:c + (1 << 28), 1]) & 0x7FFF7FFF7FFF7FFF).nonzero()[:, 0] + c
                      for c in range(0, t.shape[0], 1 << 28)])


def test_products_of_the_most_rows(ex):  # noqa: F811
    g, most = gen(4), (1 << 31) - 512
    off, w = offsets_of([most - 77, 50]), normal(g, 2, 8, 8, dtype=BF16)  # 27 rows of no expert
    at = torch.tensor([0, 1, 1 << 30, most - 300, most - 129, most - 128, most - 78, most - 77, most - 40, most - 28], device="cuda")
    x, few = torch.zeros(most, 8, dtype=BF16, device="cuda"), normal(g, 10, 8, dtype=BF16)
    x[at] = few
    out = ex.grouped_mm(x, w, off)
    assert torch.equal(nonzero_rows(out), at)
    we = w.double()[(at >= most - 77).long()]
    want, size = torch.einsum("rnk,rk->rn", we, few.double()), torch.einsum("rnk,rk->rn", we.abs(), few.double().abs())
    within(out[at], want, ULP[BF16] * want.abs() + ACC * 8 * size)
    del out
    x[most - 1] = 1  # of no expert
    dw = ex._wgrad(x, x, off)
    for j, mine in enumerate((at < most - 77, at >= most - 77)):
        v = few[mine].double()
        within(dw[j], v.T @ v, ULP[BF16] * (v.T @ v).abs() + ACC * 16 * (v.abs().T @ v.abs()))


MOST = (1 << 31) - 1  # pairs


def test_routing_of_the_longest_batch(ex):  # noqa: F811
    logits = torch.zeros(MOST, 2, dtype=BF16, device="cuda")
    logits[:, 1] = -1
    other = torch.cat([torch.tensor([0, 5, MOST - 14_000_001, MOST - 40, MOST - 1]), torch.randint(10, MOST - 50, (2000,), generator=torch.Generator().manual_seed(1))])
    other = other.unique().cuda()
    logits[other, 1] = 1
    r = ex.route_tokens(logits, 1)
    m = other.numel()
    assert r.offsets.tolist() == [0, MOST - m, MOST]
    assert torch.equal(r.pairs[MOST - m:].long(), other) and torch.equal(r.rows[MOST - m:], r.pairs[MOST - m:])
    assert (r.experts[other] == 1).all() and int(torch.count_nonzero(r.experts)) == m
    assert torch.equal(r.position[other, 0].long(), torch.arange(MOST - m, MOST, device="cuda"))
    some = torch.randint(0, MOST - m, (5000,), generator=gen(3), device="cuda")
    assert torch.equal(r.position[r.pairs[some].long(), 0].long(), some) and (r.gates[some] == 1).all()


def test_health_word_before_and_after_the_first_product():
    """A process that has launched no product does not look at the products' part of the word; one that has does."""
    script = """
import torch
from flash_sinkhorn_b200 import _lib, experts
lib = _lib.load()
torch.zeros(1, device="cuda")
assert lib.fs_device_error() == 0 and lib.fs_clear_device_error() == 0
x, w = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(2, 64, 64, dtype=torch.bfloat16, device="cuda")
off = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
usual = lib.fs_set_product_limit(0)
out = experts.grouped_mm(x, w, off)
lib.fs_set_product_limit(usual)
assert lib.fs_device_error() == 1 and bool(torch.isnan(out).all())
assert lib.fs_clear_device_error() == 0 and lib.fs_device_error() == 0
assert bool((experts.grouped_mm(x, w, off) == 64).all()) and lib.fs_device_error() == 0
"""
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]


def test_gated_act_of_large_negative_values(ex):  # noqa: F811
    """The sigmoid's relative error grows with |g| as stated, down to where it leaves the normal range and becomes 0.

    Beside it: two products and a rounding for h, three for dv; dg is s + g s (1 - s), whose terms share the error of s and differ
    by a factor of 19 or more."""
    n = 4096
    g, v, d = torch.linspace(-87.2, -20, n, device="cuda"), normal(gen(6), n, scale=3.0), normal(gen(7), n)
    g[-64:] = torch.linspace(-1000.0, -87.5, 64, device="cuda")
    u = torch.cat([g, v])[None].requires_grad_(True)
    h = ex.gated_act(u, checkpoint=False)
    (du,) = torch.autograd.grad(h, u, d[None])
    z, s = g.double(), torch.sigmoid(g.double())
    bound = 2.0**-21 + z.abs() * 2.0**-23 + 4 * 2.0**-24
    for got, want in ((h[0], z * s * v.double()), (du[0, n:], d.double() * z * s), (du[0, :n], d.double() * v.double() * s * (1 + z * (1 - s)))):
        assert ((got.double() - want).abs() <= bound * 20 / 18 * want.abs())[:-64].all()
        assert not got[-64:].any()
