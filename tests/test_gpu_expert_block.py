"""Layer norm, routing, 8-bit products, activation, sums and orthogonal updates in a row, as a block of experts uses them.

The block is compared with its definition in 64 bits on the same 8-bit codes wherever a tensor is put into 8 bits: codes are computed from what the
kernels before gave, so that a value next to a border between two codes does not count as an error. Each step's bound is the one of
its own tests.
"""
import importlib.util
import os

import pytest
import torch

from test_gpu_experts import ACC, BF16, FP32, FUN, TINY, ULP, gen, normal, within
from test_gpu_mm8 import blocks8, grouped, rows8, wide

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex():
    from flash_sinkhorn_b200 import experts
    return experts


class Block:
    """``x + experts(norm(x))``: weights, and one pass of training or (with held weights) of serving."""

    def __init__(self, ex, d, f, e, k, seed):
        g = gen(seed)
        self.ex, self.k = ex, k
        self.scale, self.shift = 1 + 0.1 * normal(g, d), 0.1 * normal(g, d)
        self.router = normal(g, e, d, scale=d**-0.5)
        self.w_in, self.w_out = normal(g, e, 2 * f, d, scale=d**-0.5, dtype=BF16), normal(g, e, d, f, scale=f**-0.5, dtype=BF16)
        self.leaves = [self.scale, self.shift, self.router, self.w_in, self.w_out]

    def held(self):
        return self.ex.to_blocks8(self.w_in), self.ex.to_blocks8(self.w_out)

    def serve(self, x, held):
        h = self.ex.layer_norm(x, self.scale, self.shift)
        r = self.ex.route_tokens(h.float() @ self.router.t(), self.k)
        return x + self.ex.expert_mlp(h, *held, r)

    def train(self, x):
        h = self.ex.layer_norm(x, self.scale, self.shift)
        r = self.ex.route_tokens(h.float() @ self.router.t(), self.k)
        u = self.ex.grouped_mm8(h, self.w_in, r, gather=True)
        a = self.ex.gated_act(u, r)
        o = self.ex.grouped_mm8(a, self.w_out, r)
        return x + self.ex.combine_rows(o, r, weighted=False), (h, r, u, a, o)


@pytest.mark.parametrize("t,d,f,e,k", [(1, 64, 48, 4, 1), (3, 200, 96, 8, 2), (300, 256, 200, 4, 2), (2000, 136, 320, 6, 3)])
def test_block(ex, t, d, f, e, k):
    b = Block(ex, d, f, e, k, t + d)
    x = normal(gen(t), t, d, dtype=BF16)
    y, (h, r, u, a, o) = b.train(x)
    ends, live = r.offsets[1:].tolist(), (r.rows >= 0)[:, None]
    n = torch.nn.functional.layer_norm(x.double(), (d,), b.scale.double(), b.shift.double())
    within(h, n, ULP[BF16] * n.abs() + 2.0**-16 * (1 + n.abs()))
    codes, scales = blocks8(b.w_in)
    want, size = grouped(rows8(h)[r.rows.long().clamp_min(0)] * live, codes * wide(scales, 2 * f, d), ends)
    within(u, want, ULP[BF16] * want.abs() + TINY[BF16] + 2.0**-15 * size)
    p = r.gates.double().reshape(-1)[r.pairs.long().clamp_min(0)][:, None] * live
    act = p * torch.nn.functional.silu(u[:, :f].double()) * u[:, f:].double()
    within(a, act, (ULP[BF16] + FUN) * act.abs() + TINY[BF16] + 2.0**-20 * (p * u[:, f:].double()).abs())
    codes, scales = blocks8(b.w_out)
    want, size = grouped(rows8(a), codes * wide(scales, d, f), ends)
    within(o, want, ULP[BF16] * want.abs() + TINY[BF16] + 2.0**-15 * size)
    back = (o.double()[r.position.long().clamp_min(0)] * (r.position >= 0)[..., None]).sum(1)
    within(y, (x.double() + back), 2 * ULP[BF16] * (x.double().abs() + 2 * back.abs()) + k * ACC * o.abs().max())
    assert torch.equal(b.serve(x, b.held()), y)  # weights held in 8 bits: the same products


@pytest.mark.parametrize("t,d,f,e,k", [(3, 96, 64, 4, 2), (700, 128, 160, 5, 2)])
def test_training_steps(ex, t, d, f, e, k):
    """Gradients reach every leaf and are the same in every run; the matrices move by an orthogonal update of them."""
    b = Block(ex, d, f, e, k, t)
    x = normal(gen(t + 1), t, d, dtype=BF16).requires_grad_()
    leaves = [x] + [v.requires_grad_() for v in b.leaves]
    dy = normal(gen(t + 2), t, d, dtype=BF16)
    grads = torch.autograd.grad(b.train(x)[0], leaves, dy)
    again = torch.autograd.grad(b.train(x)[0], leaves, dy)
    for g, h, v in zip(grads, again, leaves):
        assert g.shape == v.shape and g.dtype == v.dtype and torch.isfinite(g).all() and torch.equal(g, h) and g.abs().sum() > 0
    for g in (grads[4], grads[5]):
        m = ex.orthogonalize(g)
        used = g.abs().amax((1, 2)) > 0
        s = torch.linalg.svdvals(m[used].float())
        assert (s[:, 0] < 1.25).all() and (m[~used] == 0).all()
        # along the gradient: no update points away from it
        assert ((m.float() * g.float()).sum((1, 2))[used] > 0).all()


def test_gradient_of_the_block_follows_its_16_bit_form(ex):
    """Roundings to 8 bits are errors of 3 % or so of a value, independent of one another: gradients keep their direction."""
    t, d, f, e, k = 512, 256, 256, 4, 2
    b = Block(ex, d, f, e, k, 5)
    x = normal(gen(6), t, d, dtype=BF16).requires_grad_()
    leaves = [x] + [v.requires_grad_() for v in b.leaves]
    dy = normal(gen(7), t, d, dtype=BF16)
    y, (h, r, *_) = b.train(x)
    grads = torch.autograd.grad(y, leaves, dy)
    h = ex.layer_norm(x, b.scale, b.shift)
    r = ex.route_tokens(h.float() @ b.router.t(), k)
    ref = torch.autograd.grad(x + ex.expert_mlp(h, b.w_in, b.w_out, r, checkpoint=False), leaves, dy)
    for g, w in zip(grads, ref):
        g, w = g.double().flatten(), w.double().flatten()
        assert (g @ w) / (g.norm() * w.norm()) > 0.98


@pytest.mark.parametrize("t", [1, 2, 64, 513])
def test_serving_in_a_graph(ex, t):
    """Captured once, replayed on other inputs; a second graph of the same block beside it."""
    b = Block(ex, 192, 160, 6, 2, 9)
    held = b.held()
    xs = [normal(gen(i), t, 192, dtype=BF16) for i in range(3)]
    want = [b.serve(x, held) for x in xs]
    static = [xs[0].clone(), xs[1].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.serve(static[0], held)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(b.serve(s, held))
        graphs.append(graph)
    graphs[0].replay()
    graphs[1].replay()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    static[0].copy_(xs[2])
    graphs[0].replay()
    assert torch.equal(outs[0], want[2]) and torch.equal(outs[1], want[1])


def test_two_streams_at_once(ex):
    b = Block(ex, 256, 192, 8, 2, 11)
    held = b.held()
    xs = [normal(gen(20 + i), 400, 256, dtype=BF16) for i in range(2)]
    g = normal(gen(30), 6, 200, 180)
    want, moved = [b.serve(x, held) for x in xs], ex.orthogonalize(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got, ortho = [[], []], []
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(b.serve(xs[i], held))
        with torch.cuda.stream(streams[2]):
            ortho.append(ex.orthogonalize(g))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    assert all(torch.equal(y, moved) for y in ortho)


def test_forward_mode_derivatives_are_refused(ex):
    import torch.autograd.forward_ad as fwd
    w = torch.randn(2, 16, 32, device="cuda", dtype=BF16)
    x = torch.randn(8, 32, device="cuda", dtype=BF16)
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    with fwd.dual_level():
        dual_w, dual_x = fwd.make_dual(w, torch.ones_like(w)), fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ex.to_blocks8(dual_w), lambda: ex.orthogonalize(dual_w), lambda: ex.layer_norm(dual_x), lambda: ex.grouped_mm8(dual_x, w, off),
                     lambda: ex.grouped_mm8(x, dual_w, off)):
            with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
                call()


def test_example_runs_with_norm_and_orthogonal_updates():
    spec = importlib.util.spec_from_file_location("balanced_experts", os.path.join(ROOT, "examples", "balanced_experts.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, busiest = example.train(steps=6, tokens=512, norm=True, orthogonal=True)
    assert len(losses) == 6 and all(l == l and abs(l) < 1e6 for l in losses) and busiest >= 1.0
    torch.manual_seed(0)
    layer = example.BalancedExperts(32, 48, 4, 2, norm=True).cuda()
    y, _ = layer(torch.randn(100, 32, device="cuda"))
    y.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in layer.parameters() if p is not layer.router)
