"""The operators of routed experts (``flash_sinkhorn_b200.experts``), as a list of cases with the ranges they stand for.

``listed()`` names the cases, ``draw()`` gives further ones from the same ranges, ``prepare()`` makes what a program has
in hand before the call and ``run()`` is one pass through one operator: with ``own`` through the framework's kernels,
without it in elementary torch operations in 32 bits. ``exact()`` is the definition in 64 bits, and ``work()`` counts
what a pass cannot do without. Everything is synthetic: Gaussian activations and weights, experts of uneven popularity.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BLOCK = 32  # values that share one scale in the 8-bit checkpoint


def listed():
    return [
        # One token on its way through the first product of an expert layer (serving, batch of one): the weights of two
        # experts are read and nothing else counts.
        dict(name="mm_token", kind="mm", tokens=1, k=2, experts=16, inner=2048, outer=2048, type="bf16", skew=0.5,
             gather=True, train=False, off=0.0),
        # A decoding batch: a few rows for most experts, none for some.
        dict(name="mm_decode", kind="mm", tokens=32, k=4, experts=64, inner=2048, outer=1024, type="bf16", skew=0.8,
             gather=True, train=False, off=0.0),
        # A prompt of moderate length with odd sizes, rows that were already put in order.
        dict(name="mm_ragged_fp16", kind="mm", tokens=5003, k=1, experts=10, inner=784, outer=1100, type="fp16", skew=1.0,
             gather=False, train=False, off=0.0),
        # Long prompts, the large product: tensor cores only.
        dict(name="mm_prompt", kind="mm", tokens=8192, k=8, experts=64, inner=2048, outer=2048, type="bf16", skew=0.5,
             gather=True, train=False, off=0.0),
        # A training step's first product with both gradients; a tenth of the tokens is padding.
        dict(name="mm_train", kind="mm", tokens=8192, k=4, experts=32, inner=1024, outer=2048, type="bf16", skew=0.5,
             gather=True, train=True, off=0.1),
        # The same in a small model whose widths no vector load or tile divides.
        dict(name="mm_train_odd", kind="mm", tokens=3001, k=2, experts=7, inner=300, outer=501, type="bf16", skew=1.0,
             gather=True, train=True, off=0.0),
        # Routing of a decoding batch: launches and latency.
        dict(name="route_decode", kind="route", tokens=32, k=4, experts=64, type="bf16", bias=True, all=False, train=False,
             off=0.0),
        # Routing of a training batch with the prices of a balanced plan, and the gradient to the logits.
        dict(name="route_train", kind="route", tokens=65536, k=8, experts=128, type="fp32", bias=True, all=True, train=True,
             off=0.1),
        # The gated activation of a training step with its 8-bit checkpoint and the gradient that reads it.
        dict(name="act_train", kind="act", tokens=8192, k=4, experts=32, outer=2048, type="bf16", skew=0.5, train=True,
             off=0.0),
        # The same at a width that ends inside a block of the checkpoint.
        dict(name="act_odd", kind="act", tokens=1003, k=2, experts=8, outer=1100, type="fp16", skew=0.5, train=True,
             off=0.2),
        # Rows of the experts summed back into tokens in a training step, gate-weighted.
        dict(name="combine_train", kind="combine", tokens=16384, k=4, experts=32, inner=2048, type="bf16", skew=0.5,
             train=True, off=0.0),
        # The same for a decoding batch of an odd width.
        dict(name="combine_decode", kind="combine", tokens=37, k=4, experts=16, inner=1100, type="fp16", skew=0.5,
             train=False, off=0.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, as models have them; sometimes any number."""
    w = _log_uniform(rng, lo, hi)
    return w if rng.random() < 0.3 else max(64, w // 64 * 64)


def draw(rng):
    kind = rng.choice(["mm", "mm", "mm", "route", "act", "combine"])
    experts = _log_uniform(rng, 4, 128)
    k = rng.choice([v for v in (1, 2, 4, 6, 8) if v <= experts])
    c = dict(kind=kind, k=k, experts=experts, train=rng.random() < 0.5, off=rng.choice([0.0, 0.0, 0.1, 0.3]))
    if kind == "route":
        return dict(c, tokens=_log_uniform(rng, 1, 65536), type=rng.choice(["bf16", "fp16", "fp32", "fp32"]),
                    bias=rng.random() < 0.7, all=rng.random() < 0.5)
    c["skew"] = rng.choice([0.0, 0.5, 1.0])
    if kind == "mm":
        tokens, inner, outer = _log_uniform(rng, 1, 16384), _width(rng, 64, 2048), _width(rng, 64, 2048)
        while tokens * k > 32768 or tokens * k * float(inner) * outer > 6.8e10:
            tokens = max(1, int(tokens * rng.uniform(0.5, 0.9)))
        return dict(c, tokens=tokens, inner=inner, outer=outer, type=rng.choice(["bf16", "bf16", "fp16"]),
                    gather=rng.random() < 0.7)
    tokens, width = _log_uniform(rng, 1, 16384), _width(rng, 64, 2048)
    while tokens * k > 32768:
        tokens = max(1, int(tokens * rng.uniform(0.5, 0.9)))
    c.update(tokens=tokens, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    c["outer" if kind == "act" else "inner"] = width
    return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _uniform(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _routing(case, gen):
    """A finished routing of `tokens` tokens: k different experts each, popular ones more often, none where a token is off.

    experts, position [T, k]; offsets [E + 1]; pairs, rows [T * k] (pair and token of each row in expert order, -1 past the
    last one); gates [T, k]. `longest` is the size of the largest group, known to the host as a capacity would be.
    """
    t, k, e = case["tokens"], case["k"], case["experts"]
    popular = _normal(gen, e, scale=case["skew"])
    noise = -torch.log(-torch.log(_uniform(gen, t, e).clamp(1e-7, 1 - 1e-7)))
    experts = (popular + noise).argsort(dim=1, descending=True)[:, :k]
    gates = torch.softmax(_normal(gen, t, k), dim=1)
    on = _uniform(gen, t, 1) >= case["off"]
    experts = torch.where(on, experts, experts.new_full((), e))
    gates = torch.where(on, gates, gates.new_zeros(()))
    flat = experts.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = (flat[:, None] == torch.arange(e, device="cuda")[None, :]).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k, device="cuda")
    routed = torch.arange(t * k, device="cuda") < offsets[-1]
    pairs = torch.where(routed, order, order.new_full((), -1))
    rows = torch.where(routed, order // k, order.new_full((), -1))
    position = torch.where(flat < e, place, place.new_full((), -1)).reshape(t, k)
    experts = torch.where(experts < e, experts, experts.new_full((), -1))
    ints = {"experts": experts, "offsets": offsets, "pairs": pairs, "rows": rows, "position": position}
    return {"gates": gates, **{name: v.to(torch.int32).contiguous() for name, v in ints.items()}}, int(counts.max())


def prepare(case, seed):
    gen = _generator(seed)
    kind, train, dtype = case["kind"], case["train"], _TYPES[case["type"]]
    s = {"case": dict(case)}
    t, k, e = case["tokens"], case["k"], case["experts"]
    if kind == "route":
        # logits of a router whose experts are of uneven popularity, in the type that the router's product has
        s["logits"] = (_normal(gen, t, e) + _normal(gen, e, scale=0.5)).to(dtype).requires_grad_(train)
        s["bias"] = _normal(gen, e, scale=0.5) if case["bias"] else None
        s["mask"] = _uniform(gen, t) >= case["off"] if case["off"] > 0 else None
        s["grad"] = _normal(gen, t, k)
        return s
    s["routing"], s["longest"] = _routing(case, gen)
    if kind == "mm":
        inner, outer = case["inner"], case["outer"]
        s["x"] = _normal(gen, t if case["gather"] else t * k, inner, dtype=dtype).requires_grad_(train)
        s["w"] = _normal(gen, e, outer, inner, scale=inner**-0.5, dtype=dtype).requires_grad_(train)
        s["grad"] = _normal(gen, t * k, outer, dtype=dtype) if train else None
    elif kind == "act":
        s["u"] = _normal(gen, t * k, 2 * case["outer"], dtype=dtype).requires_grad_(train)
        s["routing"]["gates"].requires_grad_(train)
        s["grad"] = _normal(gen, t * k, case["outer"], dtype=dtype)
    else:
        s["o"] = _normal(gen, t * k, case["inner"], dtype=dtype).requires_grad_(train)
        s["routing"]["gates"].requires_grad_(train)
        s["grad"] = _normal(gen, t, case["inner"], dtype=dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------


def _pass_route(s):
    from flash_sinkhorn_b200.experts import route_tokens
    c = s["case"]
    r = route_tokens(s["logits"], c["k"], bias=s["bias"], mask=s["mask"], normalize="all" if c["all"] else "selected")
    out = [r.gates, r.experts, r.offsets, r.pairs, r.rows, r.position]
    if c["train"]:
        out += torch.autograd.grad(r.gates, (s["logits"],), s["grad"])
    return out


def _plain_route(s):
    c, l = s["case"], s["logits"].detach().float()
    t, e = l.shape
    k = c["k"]
    on = l > -math.inf
    score = l
    if s["bias"] is not None:
        score, on = score + s["bias"], on & (s["bias"] > -math.inf)
    if s["mask"] is not None:
        on = on & s["mask"][:, None]
    score = torch.where(on, score, score.new_full((), -math.inf))
    chosen = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k]
    taken = on.gather(1, chosen)
    picked = l.gather(1, chosen).masked_fill(~taken, -math.inf)
    over = l.masked_fill(~on, -math.inf) if c["all"] else picked
    top = over.amax(1, keepdim=True).clamp_min(-3e38)
    total = torch.exp(over - top).sum(1, keepdim=True)
    gates = torch.where(taken, torch.exp(picked - top) / total, picked.new_zeros(()))
    flat = torch.where(taken, chosen, chosen.new_full((), e)).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device=l.device).scatter_add_(0, flat, torch.ones_like(flat))[:e]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    here = torch.arange(t * k, device=l.device)
    place = torch.empty_like(order)
    place[order] = here
    none = order.new_full((), -1)
    pairs = torch.where(here < offsets[-1], order, none)
    rows = torch.where(here < offsets[-1], order // k, none)
    position = torch.where(flat < e, place, none).reshape(t, k)
    experts = torch.where(taken, chosen, none)
    out = [gates] + [v.to(torch.int32) for v in (experts, offsets, pairs, rows, position)]
    if c["train"]:
        inner = (gates * s["grad"]).sum(1, keepdim=True)
        direct = torch.zeros_like(l).scatter_add_(1, chosen, gates * s["grad"])
        share = torch.where(on, torch.exp(over - top) / total, l.new_zeros(())) if c["all"] else torch.zeros_like(
            l).scatter_add_(1, chosen, gates)
        out.append((direct - share * inner).to(s["logits"].dtype))
    return out


def _pass_mm(s):
    from flash_sinkhorn_b200.experts import Routing, grouped_mm
    c = s["case"]
    y = grouped_mm(s["x"], s["w"], Routing(**s["routing"]), gather=c["gather"])
    return [y, *torch.autograd.grad(y, (s["x"], s["w"]), s["grad"])] if c["train"] else [y]


def _plain_mm(s):
    c, r = s["case"], s["routing"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    n, offsets = r["pairs"].shape[0], r["offsets"].long()
    # groups padded to the longest one: [E, longest] row numbers, and whether a place holds a row
    place = offsets[:-1, None] + torch.arange(s["longest"], device=x.device)[None, :]
    held = place < offsets[1:, None]
    place = place.clamp_max(n - 1)
    source = r["rows"].long().clamp_min(0) if c["gather"] else torch.arange(n, device=x.device)
    xs = x[source[place]] * held[..., None]
    back = torch.full((n + 1,), -1, dtype=torch.int64, device=x.device)
    back[torch.where(held, place, place.new_full((), n)).reshape(-1)] = torch.arange(place.numel(), device=x.device)
    back = back[:n]

    def ordered(padded):
        rows = padded.reshape(-1, padded.shape[-1])[back.clamp_min(0)]
        return rows.masked_fill_((back < 0)[:, None], 0.0)

    out = [ordered(torch.bmm(xs, w.transpose(1, 2))).to(s["x"].dtype)]
    if c["train"]:
        dy = s["grad"].float()[place] * held[..., None]
        dx = ordered(torch.bmm(dy, w))
        if c["gather"]:
            pos = r["position"].long()
            dx = (dx[pos.clamp_min(0)] * (pos >= 0)[..., None]).sum(1)
        out += [dx.to(s["x"].dtype), torch.bmm(dy.transpose(1, 2), xs).to(s["w"].dtype)]
    return out


def _pass_act(s):
    from flash_sinkhorn_b200.experts import Routing, gated_act
    r = Routing(**s["routing"])
    h = gated_act(s["u"], r)
    return [h, *torch.autograd.grad(h, (s["u"], r.gates), s["grad"])] if s["case"]["train"] else [h]


def _held_in_8_bits(v):
    """The values that blocks of 32 stand for once they are held as an 8-bit integer each and a power of two per block:
    the smallest one at which the block's largest magnitude rounds to 127 at most."""
    n, f = v.shape
    b = torch.nn.functional.pad(v, (0, -f % _BLOCK)).reshape(n, -1, _BLOCK)
    m, p = torch.frexp(b.abs().amax(2, keepdim=True))
    scale = torch.ldexp(torch.ones_like(m), torch.where(m < 127.5 / 128, p - 7, p - 6).clamp_min(-126))
    return (torch.round(b / scale) * scale).reshape(n, -1)[:, :f]


def _plain_act(s):
    r, f = s["routing"], s["case"]["outer"]
    u, pairs = s["u"].detach().float(), r["pairs"].long()
    gate = torch.where(pairs >= 0, r["gates"].detach().reshape(-1)[pairs.clamp_min(0)], 0.0)[:, None]
    g, v = u[:, :f], u[:, f:]
    h = (gate * g * torch.sigmoid(g) * v).to(s["u"].dtype)
    if not s["case"]["train"]:
        return [h]
    dh = s["grad"].float()
    g, v = _held_in_8_bits(g), _held_in_8_bits(v)
    sig = torch.sigmoid(g)
    du = torch.cat([gate * dh * v * sig * (1 + g * (1 - sig)), gate * dh * g * sig], dim=1)
    dgate = torch.zeros(r["gates"].numel() + 1, device=u.device)
    dgate[torch.where(pairs >= 0, pairs, r["gates"].numel())] = (dh * g * sig * v).sum(1)
    return [h, du.to(s["u"].dtype), dgate[:-1].reshape(r["gates"].shape)]


def _pass_combine(s):
    from flash_sinkhorn_b200.experts import Routing, combine_rows
    r = Routing(**s["routing"])
    y = combine_rows(s["o"], r)
    return [y, *torch.autograd.grad(y, (s["o"], r.gates), s["grad"])] if s["case"]["train"] else [y]


def _plain_combine(s):
    r, o = s["routing"], s["o"].detach().float()
    gates, pos = r["gates"].detach(), r["position"].long()
    rows = o[pos.clamp_min(0)] * (pos >= 0)[..., None]
    y = (gates[..., None] * rows).sum(1)
    out = [y.to(s["o"].dtype)]
    if s["case"]["train"]:
        dy, pairs = s["grad"].float(), r["pairs"].long().clamp_min(0)
        weight = torch.where(r["pairs"] >= 0, gates.reshape(-1)[pairs], 0.0)
        do = weight[:, None] * dy[pairs // pos.shape[1]]
        out += [do.to(s["o"].dtype), (rows * dy[:, None, :]).sum(2)]
    return out


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"route": _pass_route, "mm": _pass_mm, "act": _pass_act, "combine": _pass_combine}[kind](s)
    return {"route": _plain_route, "mm": _plain_mm, "act": _plain_act, "combine": _plain_combine}[kind](s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    kind, b, train = case["kind"], _BYTES[case["type"]], case["train"]
    t, k, e = case["tokens"], case["k"], case["experts"]
    pairs = t * k
    routed = pairs * (1 - case["off"])
    if kind == "route":
        # logits in; gate, expert and position of each pair, pair and row in order, offsets out. Backward: the experts and
        # gates (or all logits again) and the gradient in, a gradient for every logit out.
        n = t * e * b + pairs * 20 + (e + 1) * 4
        if train:
            n += t * e * b + pairs * 12 + (t * e * b if case["all"] else 0)
        return {"bytes": n, "flops": t * e * (8 if train else 4)}
    if kind == "mm":
        inner, outer = case["inner"], case["outer"]
        used = e * (1 - (1 - 1 / e) ** max(1.0, routed)) if pairs < 8 * e else e  # experts that have rows
        x = (t if case["gather"] else pairs) * inner * b
        n = x + used * inner * outer * b + pairs * outer * b
        if train:
            n += x + pairs * outer * b + used * inner * outer * b + x + e * inner * outer * b
        return {"bytes": n, "flops": 2.0 * routed * inner * outer * (3 if train else 1)}
    if kind == "act":
        f = case["outer"]
        n = pairs * f * b * 3 + pairs * 8
        if train:  # the checkpoint is written and read: a byte for each value, and one for each block
            n += pairs * 2 * (2 * f + 2 * -(-f // _BLOCK)) + pairs * f * b * 3 + pairs * 8
        return {"bytes": n, "flops": pairs * f * (30.0 if train else 8.0)}
    d = case["inner"]
    n = routed * d * b + t * d * b + pairs * 8
    if train:
        n += routed * d * b + t * d * b + pairs * d * b + pairs * 12
    return {"bytes": n, "flops": pairs * d * (6.0 if train else 2.0)}


# ---------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "mm": _exact_mm, "act": _exact_act, "combine": _exact_combine}[case["kind"]](s)


def _exact_route(s):
    """Gates and their gradient; the selection itself is of 32-bit scores, so it is taken from those."""
    c = s["case"]
    l = s["logits"].detach()
    on = torch.isfinite(l) if s["mask"] is None else torch.isfinite(l) & s["mask"][:, None]
    score = l.float() if s["bias"] is None else l.float() + s["bias"]
    left = torch.where(on, score, float("-inf")).clone()
    picks, token = [], torch.arange(l.shape[0], device=l.device)
    for _ in range(c["k"]):
        best = left.max(1, keepdim=True).values
        first = (left == best).to(torch.int8).argmax(1)  # the first of the largest
        picks.append(first)
        left[token, first] = float("-inf")
    chosen = torch.stack(picks, 1)
    z = l.double()
    if c["all"]:
        z = z.masked_fill(~on, float("-inf"))
        p = torch.nan_to_num(torch.softmax(z, 1))
        gates = p.gather(1, chosen)
    else:
        live = on.gather(1, chosen)
        gates = torch.nan_to_num(torch.softmax(z.gather(1, chosen).masked_fill(~live, float("-inf")), 1))
    out = [gates, None, None, None, None, None]
    if c["train"]:
        dg = s["grad"].double()
        if c["all"]:  # d gate_s / d logit_j = p_s (delta_sj - p_j)
            dl = -p * (gates * dg).sum(1, keepdim=True)
        else:
            dl = torch.zeros_like(z).scatter_add(1, chosen, -gates * (gates * dg).sum(1, keepdim=True))
        out.append(dl.scatter_add(1, chosen, gates * dg))
    return out


def _exact_mm(s):
    c, r = s["case"], s["routing"]
    x, w = s["x"].detach(), s["w"].detach()
    n, ends = r["pairs"].shape[0], r["offsets"].tolist()
    y = torch.zeros(n, c["outer"], dtype=torch.float64, device=x.device)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device) if c["train"] else None
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        if lo == hi:
            continue
        index = r["rows"][lo:hi].long() if c["gather"] else torch.arange(lo, hi, device=x.device)
        a, we = x[index].double(), w[e].double()
        y[lo:hi] = a @ we.T
        if c["train"]:
            dy = s["grad"][lo:hi].double()
            dx.index_add_(0, index, dy @ we)
            dw[e] = dy.T @ a
    return [y, dx, dw] if c["train"] else [y]


def _exact_act(s):
    c, r = s["case"], s["routing"]
    f, u, pairs = c["outer"], s["u"].detach().double(), r["pairs"].long()
    routed = (pairs >= 0).double()
    p = (r["gates"].detach().double().reshape(-1)[pairs.clamp_min(0)] * routed)[:, None]
    h = p * torch.nn.functional.silu(u[:, :f]) * u[:, f:]
    if not c["train"]:
        return [h]
    halves = []
    for half in (u[:, :f], u[:, f:]):
        q = torch.empty_like(half)
        for at in range(0, f, _BLOCK):
            b = half[:, at:at + _BLOCK]
            top = b.abs().amax(1, keepdim=True).clamp_min(2.0**-126)
            step = torch.exp2(torch.floor(torch.log2(top)) - 6)
            step = torch.where(torch.round(top / step) > 127, 2 * step, step)
            q[:, at:at + _BLOCK] = torch.round(b / step) * step
        halves.append(q)
    g, v = halves
    dh, sig = s["grad"].double(), torch.sigmoid(g)
    du = torch.cat([p * dh * v * (sig + g * sig * (1 - sig)), p * dh * g * sig], 1)
    dp = torch.zeros(r["gates"].numel(), dtype=torch.float64, device=u.device)
    dp.index_add_(0, pairs.clamp_min(0), routed * (dh * g * sig * v).sum(1))
    return [h, du, dp.reshape(r["gates"].shape)]


def _exact_combine(s):
    c, r = s["case"], s["routing"]
    o, gates = s["o"].detach().double(), r["gates"].detach().double()
    pairs, k = r["pairs"].long(), c["k"]
    routed = pairs >= 0
    at, row = pairs[routed], torch.nonzero(routed)[:, 0]
    y = torch.zeros(c["tokens"], c["inner"], dtype=torch.float64, device=o.device)
    y.index_add_(0, at // k, gates.reshape(-1)[at, None] * o[row])
    if not c["train"]:
        return [y]
    dy = s["grad"].double()
    do = torch.zeros_like(o)
    do[row] = gates.reshape(-1)[at, None] * dy[at // k]
    dgate = torch.zeros(gates.numel(), dtype=torch.float64, device=o.device)
    dgate[at] = (o[row] * dy[at // k]).sum(1)
    return [y, do, dgate.reshape(gates.shape)]
