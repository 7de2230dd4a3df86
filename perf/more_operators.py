"""What stands around routed experts (``flash_sinkhorn_b200.experts``): the layer norm before them, their products in 8-bit
floating point, and the orthogonal update of their weights, as a list of cases with the ranges they stand for.

``listed()`` names the cases, ``draw()`` gives further ones from the same ranges, ``prepare()`` makes what a program has
in hand before the call and ``run()`` is one pass through one operator: with ``own`` through the framework's kernels,
without it in elementary torch operations in 32 bits. ``exact()`` is the definition in 64 bits, and ``work()`` counts
what a pass cannot do without. Everything is synthetic.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BLOCK = 128  # values, or rows and columns of a weight, that share one scale
_TOP = 448.0  # largest value of the 8-bit type (4 bits of exponent, 3 of mantissa)
_STEPS, _A, _B, _C = 5, 3.4445, -4.7750, 2.0315  # x -> A x + B x^3 + C x^5 on the singular values


def listed():
    return [
        # The norm before a layer while a batch is decoded: one launch and its latency.
        dict(name="norm_decode", kind="norm", rows=32, width=2048, type="bf16", weights="fp32", train=False),
        # A training step's norm, forward and backward, with the sums over all rows for weight and bias.
        dict(name="norm_train", kind="norm", rows=16384, width=2048, type="bf16", weights="fp32", train=True),
        # The same where no vector load divides the rows, in 32 bits.
        dict(name="norm_odd", kind="norm", rows=3001, width=501, type="fp32", weights="fp32", train=True),
        # Few, very long rows, weights of the rows' type.
        dict(name="norm_wide", kind="norm", rows=512, width=16384, type="fp16", weights="fp16", train=True),
        # One token through a product whose weights are held in 8 bits (serving, batch of one).
        dict(name="mm_token", kind="mm", tokens=1, k=2, experts=16, inner=2048, outer=2048, type="bf16", skew=0.5,
             gather=True, held=True, train=False, off=0.0),
        # A decoding batch: a few rows for most experts, none for some.
        dict(name="mm_decode", kind="mm", tokens=32, k=4, experts=64, inner=2048, outer=1024, type="bf16", skew=0.8,
             gather=True, held=True, train=False, off=0.0),
        # Long prompts: tensor cores only.
        dict(name="mm_prompt", kind="mm", tokens=8192, k=8, experts=64, inner=2048, outer=2048, type="bf16", skew=0.5,
             gather=True, held=True, train=False, off=0.0),
        # A training step: rows and weights are put into 8 bits anew, both gradients; a tenth of the tokens is padding.
        dict(name="mm_train", kind="mm", tokens=8192, k=4, experts=32, inner=1024, outer=2048, type="bf16", skew=0.5,
             gather=True, held=False, train=True, off=0.1),
        # The same in a small model whose widths end inside of blocks, rows already in order.
        dict(name="mm_odd", kind="mm", tokens=3001, k=2, experts=7, inner=300, outer=501, type="fp16", skew=1.0,
             gather=False, held=False, train=True, off=0.0),
        # The update of one small matrix: a chain of small products, so launches and latency.
        dict(name="ortho_small", kind="ortho", count=1, rows=512, cols=512, type="fp32"),
        # The update of a layer of experts: tensor cores only.
        dict(name="ortho_experts", kind="ortho", count=32, rows=2048, cols=1024, type="bf16"),
        # The same for odd sizes, more columns than rows.
        dict(name="ortho_odd", kind="ortho", count=7, rows=300, cols=501, type="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, as models have them; sometimes any number."""
    w = _log_uniform(rng, lo, hi)
    return w if rng.random() < 0.3 else max(64, w // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "mm", "mm", "ortho"])
    if kind == "norm":
        rows, width, dtype = _log_uniform(rng, 1, 65536), _width(rng, 64, 16384), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        while rows * width > 16384 * 2048:
            rows = max(1, int(rows * rng.uniform(0.3, 0.9)))
        return dict(kind=kind, rows=rows, width=width, type=dtype, weights=rng.choice(["fp32", dtype]), train=rng.random() < 0.6)
    if kind == "mm":
        experts = _log_uniform(rng, 1, 128)
        k = rng.choice([v for v in (1, 2, 4, 6, 8) if v <= experts])
        tokens, inner, outer = _log_uniform(rng, 1, 16384), _width(rng, 64, 2048), _width(rng, 64, 2048)
        while tokens * k > 32768 or tokens * k * float(inner) * outer > 6.8e10:
            tokens = max(1, int(tokens * rng.uniform(0.5, 0.9)))
        train = rng.random() < 0.4
        return dict(kind=kind, tokens=tokens, k=k, experts=experts, inner=inner, outer=outer, type=rng.choice(["bf16", "bf16", "fp16"]),
                    skew=rng.choice([0.0, 0.5, 1.0]), gather=rng.random() < 0.7, held=not train, train=train,
                    off=rng.choice([0.0, 0.0, 0.1, 0.3]))
    rows, cols, count = _width(rng, 64, 2048), _width(rng, 64, 2048), _log_uniform(rng, 1, 32)
    while count > 1 and count * float(rows) * cols * min(rows, cols) > 6.8e10:
        count = max(1, int(count * rng.uniform(0.5, 0.9)))
    return dict(kind=kind, count=count, rows=rows, cols=cols, type=rng.choice(["bf16", "fp16", "fp32"]))


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _routing(case, gen):
    """A finished routing of `tokens` tokens: k different experts each, popular ones more often, none where a token is off.

    The fields of a ``Routing``, and `longest`, the size of the largest group, known to the host as a capacity would be.
    """
    t, k, e = case["tokens"], case["k"], case["experts"]
    dev = "cuda"
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=gen, device=dev).clamp(1e-7, 1 - 1e-7)))
    chosen = (_normal(gen, e, scale=case["skew"]) + noise).argsort(dim=1, descending=True)[:, :k]
    gates = torch.softmax(_normal(gen, t, k), dim=1)
    on = torch.rand(t, 1, generator=gen, device=dev) >= case["off"]
    chosen = chosen.where(on, chosen.new_full((), e))
    gates = gates.where(on, gates.new_zeros(()))
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = (flat[:, None] == torch.arange(e, device=dev)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    here, none = torch.arange(t * k, device=dev), order.new_full((), -1)
    place = torch.empty_like(order)
    place[order] = here
    routed = here < offsets[-1]
    ints = {"experts": chosen.where(chosen < e, none), "offsets": offsets, "pairs": order.where(routed, none),
            "rows": (order // k).where(routed, none), "position": place.where(flat < e, none).reshape(t, k)}
    return {"gates": gates, **{name: v.to(torch.int32).contiguous() for name, v in ints.items()}}, int(counts.max())


def _scale_of(top):
    """The smallest power of two (from 2^-126 on) by which values up to `top` are divided to fit the 8-bit type."""
    m, p = torch.frexp(top)
    return torch.ldexp(torch.ones_like(m), torch.where(m > _TOP / 512, p - 8, p - 9).clamp_min(-126))


def _blocks_of_weights(w):
    """8-bit codes and scales of w [E, N, K]: one scale for 128 x 128 values."""
    e, n, k = w.shape
    b = torch.nn.functional.pad(w.float(), (0, -k % _BLOCK, 0, -n % _BLOCK))
    b = b.reshape(e, -(-n // _BLOCK), _BLOCK, -(-k // _BLOCK), _BLOCK)
    scale = _scale_of(b.abs().amax((2, 4)))
    codes = (b / scale[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return codes.reshape(e, n + -n % _BLOCK, k + -k % _BLOCK)[:, :n, :k], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], _TYPES[case["type"]]
    s = {"case": dict(case)}
    if kind == "norm":
        rows, width, train = case["rows"], case["width"], case["train"]
        # a residual stream: some features are far larger than others, and the mean is not zero
        size = torch.exp(0.5 * _normal(gen, width))
        s["x"] = (_normal(gen, rows, width) * size + 0.3 * _normal(gen, rows, 1)).to(dtype).requires_grad_(train)
        s["w"] = (1 + _normal(gen, width, scale=0.2)).to(_TYPES[case["weights"]]).requires_grad_(train)
        s["b"] = _normal(gen, width, scale=0.2, dtype=_TYPES[case["weights"]]).requires_grad_(train)
        s["grad"] = _normal(gen, rows, width, dtype=dtype) if train else None
    elif kind == "mm":
        t, k, e, inner, outer, train = (case[v] for v in ("tokens", "k", "experts", "inner", "outer", "train"))
        s["routing"], s["longest"] = _routing(case, gen)
        s["x"] = _normal(gen, t if case["gather"] else t * k, inner, dtype=dtype).requires_grad_(train)
        w = _normal(gen, e, outer, inner, scale=inner**-0.5, dtype=dtype)
        if case["held"]:  # rows a multiple of 16 bytes apart, as a program keeps them
            codes, s["scales"] = _blocks_of_weights(w)
            s["codes"] = torch.zeros(e, outer, inner + -inner % 16, dtype=codes.dtype, device="cuda")[:, :, :inner]
            s["codes"].copy_(codes)
        else:
            s["w"] = w.requires_grad_(train)
        s["grad"] = _normal(gen, t * k, outer, dtype=dtype) if train else None
    else:
        n, rows, cols = case["count"], case["rows"], case["cols"]
        # a momentum: some strong directions over noise, of a gradient's small magnitude
        r = max(1, min(rows, cols) // 4)
        strong = torch.logspace(0, -2, r, device="cuda")
        s["g"] = (1e-3 * ((_normal(gen, n, rows, r) * strong) @ _normal(gen, n, r, cols) + 0.1 * _normal(gen, n, rows, cols))).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------


def _pass_norm(s):
    from flash_sinkhorn_b200.experts import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"])
    return [y, *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["grad"])] if s["case"]["train"] else [y]


def _plain_norm(s):
    x, w, b = (s[v].detach().float() for v in ("x", "w", "b"))
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-5)
    n = d * r
    out = [(n * w + b).to(s["x"].dtype)]
    if s["case"]["train"]:
        g = s["grad"].float()
        u = g * w
        dx = r * (u - u.mean(1, keepdim=True) - n * (u * n).mean(1, keepdim=True))
        out += [dx.to(s["x"].dtype), (g * n).sum(0).to(s["w"].dtype), g.sum(0).to(s["b"].dtype)]
    return out


def _pass_mm(s):
    from flash_sinkhorn_b200.experts import Blocks8, Routing, grouped_mm8
    c = s["case"]
    w = Blocks8(s["codes"], s["scales"]) if c["held"] else s["w"]
    y = grouped_mm8(s["x"], w, Routing(**s["routing"]), gather=c["gather"])
    return [y, *torch.autograd.grad(y, (s["x"], s["w"]), s["grad"])] if c["train"] else [y]


def _rows_in_8_bits(v):
    """The values that rows stand for once blocks of 128 of them are held in 8 bits each, with a scale per block."""
    n, f = v.shape
    b = torch.nn.functional.pad(v, (0, -f % _BLOCK)).reshape(n, -1, _BLOCK)
    scale = _scale_of(b.abs().amax(2, keepdim=True))
    return ((b / scale).to(torch.float8_e4m3fn).float() * scale).reshape(n, -1)[:, :f]


def _plain_mm(s):
    c, r = s["case"], s["routing"]
    x = s["x"].detach().float()
    codes, scales = (s["codes"], s["scales"]) if c["held"] else _blocks_of_weights(s["w"].detach())
    wide = scales.repeat_interleave(_BLOCK, 1)[:, :c["outer"]].repeat_interleave(_BLOCK, 2)[:, :, :c["inner"]]
    w = codes.float() * wide
    n, offsets = r["pairs"].shape[0], r["offsets"].long()
    # groups padded to the longest one: [E, longest] row numbers, and whether a place holds a row
    place = offsets[:-1, None] + torch.arange(s["longest"], device=x.device)
    held = place < offsets[1:, None]
    place = place.clamp_max(n - 1)
    source = r["rows"].long().clamp_min(0)[place] if c["gather"] else place
    back = torch.full((n + 1,), -1, dtype=torch.int64, device=x.device)
    back[torch.where(held, place, place.new_full((), n)).reshape(-1)] = torch.arange(place.numel(), device=x.device)
    back = back[:n]

    def ordered(padded):
        return padded.reshape(-1, padded.shape[-1])[back.clamp_min(0)].masked_fill_((back < 0)[:, None], 0.0)

    out = [ordered(torch.bmm(_rows_in_8_bits(x)[source] * held[..., None], w.transpose(1, 2))).to(s["x"].dtype)]
    if c["train"]:
        g = s["grad"].float()
        dx = ordered(torch.bmm(_rows_in_8_bits(g)[place] * held[..., None], w))
        if c["gather"]:
            pos = r["position"].long()
            dx = (dx[pos.clamp_min(0)] * (pos >= 0)[..., None]).sum(1)
        dw = torch.bmm((g[place] * held[..., None]).transpose(1, 2), x[source] * held[..., None])
        out += [dx.to(s["x"].dtype), dw.to(s["w"].dtype)]
    return out


def _pass_ortho(s):
    from flash_sinkhorn_b200.experts import orthogonalize
    return [orthogonalize(s["g"])]


def _plain_ortho(s):
    x = s["g"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    for _ in range(_STEPS):
        a = torch.bmm(x, x.transpose(1, 2))
        x = _A * x + torch.bmm(_B * a + _C * torch.bmm(a, a), x)
    return [(x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()]


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"norm": _pass_norm, "mm": _pass_mm, "ortho": _pass_ortho}[kind](s)
    return {"norm": _plain_norm, "mm": _plain_mm, "ortho": _plain_ortho}[kind](s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    kind, b = case["kind"], _BYTES[case["type"]]
    if kind == "norm":
        n, width, bw = case["rows"] * case["width"], case["width"], _BYTES[case["weights"]]
        # x in, y out; backward: x and the gradient in, the gradient to x out, those of weight and bias out
        total = 2 * n * b + 2 * width * bw
        if case["train"]:
            total += 3 * n * b + 3 * width * bw
        return {"bytes": total, "flops": n * (19.0 if case["train"] else 8.0)}
    if kind == "mm":
        t, k, e, inner, outer = (case[v] for v in ("tokens", "k", "experts", "inner", "outer"))
        pairs = t * k
        routed = pairs * (1 - case["off"])
        used = e * (1 - (1 - 1 / e) ** max(1.0, routed)) if pairs < 8 * e else e  # experts that have rows
        x = (t if case["gather"] else pairs) * inner * b
        n = x + used * inner * outer * (1 if case["held"] else b) + pairs * outer * b
        if case["train"]:  # the weights' codes once more; rows and gradient in, both gradients out
            n += x + pairs * outer * b + used * inner * outer + x + e * inner * outer * b
        return {"bytes": n, "flops": 2.0 * routed * inner * outer * (3 if case["train"] else 1)}
    n, rows, cols = case["count"], case["rows"], case["cols"]
    m, k = min(rows, cols), max(rows, cols)
    # of the symmetric products one half; x^T x, its square, and the product with x in every step
    return {"bytes": n * rows * cols * (b + 2), "flops": _STEPS * n * (float(m) * m * k + float(m) * m * m + 2.0 * m * m * k)}


# ---------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "mm": _exact_mm, "ortho": _exact_ortho}[case["kind"]](s)


def _exact_norm(s):
    x, w, b = (s[v].detach().double() for v in ("x", "w", "b"))
    width = x.shape[1]
    sd = torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
    hat = (x - x.mean(1, keepdim=True)) / sd
    y = torch.addcmul(b.expand_as(x), hat, w)
    if not s["case"]["train"]:
        return [y]
    g = s["grad"].double()
    dhat = g * w
    dx = (width * dhat - dhat.sum(1, keepdim=True) - hat * (dhat * hat).sum(1, keepdim=True)) / (width * sd)
    return [y, dx, torch.einsum("rf,rf->f", g, hat), torch.einsum("rf->f", g)]


def _round_8(v, over):
    """Values v [..] with the largest magnitudes `over` of their blocks, as the 8-bit type holds them, in 64 bits."""
    over = over.clamp_min(_TOP * 2.0**-126)
    scale = torch.exp2(torch.ceil(torch.log2(over / _TOP)))
    scale = torch.where(over / scale > _TOP, scale * 2, torch.where(over / scale * 2 <= _TOP, scale / 2, scale))
    q = v / scale
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0**-6))) - 3)  # 3 bits of mantissa; subnormals in steps of 2^-9
    return torch.round(q / step) * step * scale


def _exact_rows(v):
    out = torch.empty_like(v)
    for at in range(0, v.shape[1], _BLOCK):
        b = v[:, at:at + _BLOCK]
        out[:, at:at + _BLOCK] = _round_8(b, b.abs().amax(1, keepdim=True))
    return out


def _exact_mm(s):
    c, r = s["case"], s["routing"]
    x = s["x"].detach().double()
    n, ends = r["pairs"].shape[0], r["offsets"].tolist()
    q = _exact_rows(x)
    y = torch.zeros(n, c["outer"], dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw = torch.zeros(c["experts"], c["outer"], c["inner"], dtype=torch.float64, device=x.device) if c["train"] else None
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        if lo == hi:
            continue
        w = torch.empty(c["outer"], c["inner"], dtype=torch.float64, device=x.device)
        for i in range(0, c["outer"], _BLOCK):
            for j in range(0, c["inner"], _BLOCK):
                at = (slice(i, i + _BLOCK), slice(j, j + _BLOCK))
                if c["held"]:
                    w[at] = s["codes"][e][at].double() * s["scales"][e, i // _BLOCK, j // _BLOCK].double()
                else:
                    b = s["w"].detach()[e][at].double()
                    w[at] = _round_8(b, b.abs().max())
        index = r["rows"][lo:hi].long() if c["gather"] else torch.arange(lo, hi, device=x.device)
        y[lo:hi] = q[index] @ w.T
        if c["train"]:
            g = s["grad"][lo:hi].double()
            dx.index_add_(0, index, _exact_rows(g) @ w)
            dw[e] = g.T @ x[index]
    return [y, dx, dw] if c["train"] else [y]


def _exact_ortho(s):
    """One matrix at a time, by the powers of g g^T or g^T g, whichever is smaller."""
    if s["case"]["count"] * float(s["case"]["rows"]) * s["case"]["cols"] > 1.4e8:
        return None
    out = []
    for g in s["g"].double().unbind(0):
        x = g / (torch.linalg.vector_norm(g) + 1e-7)
        for _ in range(_STEPS):
            if x.shape[0] <= x.shape[1]:
                h = x @ x.T
                x = _A * x + _B * (h @ x) + _C * (h @ (h @ x))
            else:
                h = x.T @ x
                x = _A * x + _B * (x @ h) + _C * ((x @ h) @ h)
        out.append(x)
    return [torch.stack(out)]
