"""Routed experts, balanced by entropic transport: the operators between a router and its tokens.

Tokens and the rows of a router are two clouds, and a plan between them with uniform marginals sends the same share of
tokens to every expert. Since ``|x - w|^2 / 2 = |x|^2 / 2 + |w|^2 / 2 - x.w``, the plan of the framework's solver is
largest where ``x.w_e + bias_e`` is, with one price per expert: :func:`transport_bias`. What uses the prices is here:

* :func:`route_tokens` - the k experts of every token, their gates, and the order of the rows (:class:`Routing`);
* :func:`grouped_mm` - the experts' matrix products over groups of any size, one row or thousands;
* :func:`gated_act` - ``gate * silu(g) * v``, with its input kept in 8 bits for the backward pass;
* :func:`combine_rows` - the experts' rows summed back into tokens;
* :func:`expert_mlp` - the three in a row, as one layer with one backward pass.

All of it runs on the current stream of the tensors' device, never waits for the host (group sizes stay on the device, so
a call can be captured in a CUDA graph), and gives the same bits in every run. Sums are held in fp32. Extension without a
counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from flash_sinkhorn_b200 import _lib

__all__ = ["Routing", "route_tokens", "grouped_mm", "gated_act", "combine_rows", "expert_mlp", "transport_bias"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BLOCK = 32  # values of the 8-bit checkpoint that share a scale
MAX_EXPERTS = 1024
MAX_K = 32


class Routing(NamedTuple):
    """Where the rows of ``T`` tokens and ``k`` slots go; row ``i`` of a grouped tensor belongs to pair ``pairs[i]``."""

    gates: torch.Tensor  #: ``[T, k]`` float32, 0 for a slot without an expert; differentiable
    experts: torch.Tensor  #: ``[T, k]`` int32, -1 for a slot without an expert
    offsets: torch.Tensor  #: ``[E + 1]`` int32; expert e has rows ``offsets[e]`` to ``offsets[e + 1]``
    pairs: torch.Tensor  #: ``[T * k]`` int32 pair (``token * k + slot``) of each row, -1 after the last routed one
    rows: torch.Tensor  #: ``[T * k]`` int32 token of each row, -1 after the last routed one
    position: torch.Tensor  #: ``[T, k]`` int32 row of each pair, -1 for a slot without an expert


def _check_type(name: str, t: torch.Tensor, types=tuple(_TYPES)) -> None:
    if t.dtype not in types:
        raise ValueError(f"{name} must be of type {', '.join(str(d).split('.')[-1] for d in types)}, got {t.dtype}")


def _device_of(name: str, t: torch.Tensor, **others: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor.")
    dev = t.device
    for other, v in others.items():
        if v.device != dev:
            raise ValueError(f"{other} must be on the same CUDA device as {name} ({dev}), got {v.device}")
    return dev


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its rows are contiguous and do not overlap, else a copy."""
    ld, one = t.stride()
    return t if one == 1 and ld >= t.shape[1] else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    ld, width = t.stride(0), t.shape[1]
    return ld if ld > width else width  # the stride of a single row says nothing


def _check_routing(r: Routing, device: torch.device, *used: str) -> None:
    """The fields ``used`` have the types, shapes and places that the kernels count on."""
    if not isinstance(r, Routing):
        raise ValueError(f"routing must be a Routing, got {type(r).__name__}")
    shape = r.position.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"routing.position must be of shape (T, k), got {tuple(shape)}")
    for name in used:
        v = getattr(r, name)
        want = torch.float32 if name == "gates" else torch.int32
        fits = v.shape == shape if name in ("gates", "experts", "position") else (
            v.ndim == 1 and (v.shape[0] == shape[0] * shape[1] if name != "offsets" else v.shape[0] > 1))
        if not fits or v.dtype != want or v.device != device or not v.is_contiguous():
            raise ValueError(f"routing.{name} must be a contiguous {want} tensor on {device} that fits {tuple(shape)} "
                             f"(tokens, slots), got {v.dtype} {tuple(v.shape)} on {v.device}")


def _check_offsets(offsets: torch.Tensor, device: torch.device) -> None:
    if offsets.ndim != 1 or offsets.dtype != torch.int32 or not offsets.is_contiguous() or offsets.device != device or len(
            offsets) < 2:
        raise ValueError(f"offsets must be a contiguous int32 tensor of shape (E + 1,) on {device}")


# ---------------------------------------------------------------------------------------------------------------
# Routing
# ---------------------------------------------------------------------------------------------------------------


def _route(logits, k, bias, mask, over_all):
    dev, (t, e) = logits.device, logits.shape
    n = t * k
    gates = torch.empty((t, k), dtype=torch.float32, device=dev)
    nbytes = _lib.load().fs_route_bytes(t, e, k)
    whole = torch.empty(4 * n + e + 1 + nbytes // 4, dtype=torch.int32, device=dev)  # with the scratch at its end
    experts, position = whole[:2 * n].view(2, t, k).unbind()
    pairs, rows = whole[2 * n:4 * n].view(2, n).unbind()
    offsets = whole[4 * n:4 * n + e + 1]
    at = whole.data_ptr()
    _lib.call("fs_route", dev, logits.data_ptr(), _TYPES[logits.dtype], _ld(logits), t, e, k, _lib.ptr(bias), _lib.ptr(mask),
              over_all, gates.data_ptr(), at, at + 16 * n, at + 8 * n, at + 12 * n, at + 4 * n, at + 16 * n + 4 * (e + 1), nbytes,
              _lib.stream_ptr(dev))
    return gates, experts, offsets, pairs, rows, position


class _RouteFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, bias, mask, over_all):
        gates, *ints = _route(logits, k, bias, mask, over_all)
        ctx.save_for_backward(logits, bias, mask, gates, ints[0])
        ctx.over_all = over_all
        ctx.mark_non_differentiable(*ints)
        return (gates, *ints)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        logits, bias, mask, gates, experts = ctx.saved_tensors
        t, e = logits.shape
        grad = grad.contiguous()
        out = torch.empty((t, e), dtype=logits.dtype, device=logits.device)
        _lib.call("fs_route_grad", logits.device, _lib.ptr(logits), _TYPES[logits.dtype], _ld(logits), t, e, gates.shape[1],
                  _lib.ptr(bias), _lib.ptr(mask), int(ctx.over_all), _lib.ptr(gates), _lib.ptr(experts), _lib.ptr(grad),
                  _lib.ptr(out), _lib.stream_ptr(logits.device))
        return out, None, None, None, None


def route_tokens(logits: torch.Tensor, k: int, *, bias: Optional[torch.Tensor] = None,
                 mask: Optional[torch.Tensor] = None, normalize: str = "selected") -> Routing:
    """Chooses ``k`` experts for every row of ``logits [T, E]`` and puts the pairs in the order of the experts.

    The chosen ones have the largest ``logits + bias`` (in fp32; ties go to the lower expert, NaN comes first so that it
    shows in the gates); ``bias [E]``, for instance prices of :func:`transport_bias`, only takes part in the choice.
    Experts whose logit or bias is ``-inf``, and all experts of tokens whose ``mask [T]`` is False, are never chosen. Gates
    are the soft-max of the logits over the chosen experts (``normalize="selected"``) or over all experts that can be
    chosen (``"all"``), and carry the gradient to ``logits`` (fp32, fp16 or bf16).
    """
    if logits.ndim != 2:
        raise ValueError(f"logits must be 2D [T, E], got shape {tuple(logits.shape)}")
    _check_type("logits", logits)
    t, e = logits.shape
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"the number of experts must be between 1 and {MAX_EXPERTS}, got {e}")
    if not 1 <= int(k) <= min(e, MAX_K):
        raise ValueError(f"k must be between 1 and {min(e, MAX_K)}, got {k}")
    if normalize not in ("selected", "all"):
        raise ValueError(f"normalize must be 'selected' or 'all', got {normalize!r}")
    _device_of("logits", logits)
    if bias is not None:
        _device_of("logits", logits, bias=bias)
        if bias.shape != (e,):
            raise ValueError(f"bias must have shape ({e},), got {tuple(bias.shape)}")
        if bias.requires_grad:
            raise ValueError("bias must not require grad (it only takes part in the choice)")
        bias = _lib.f32c(bias)
    if mask is not None:
        _device_of("logits", logits, mask=mask)
        if mask.shape != (t,) or mask.dtype != torch.bool:
            raise ValueError(f"mask must be a bool tensor of shape ({t},), got {mask.dtype} {tuple(mask.shape)}")
        mask = mask.contiguous()
    if t * int(k) >= 1 << 31:
        raise ValueError("T * k must be below 2^31")
    if t and e:
        logits = _rows_of(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return Routing(*_RouteFunction.apply(logits, int(k), bias, mask, normalize == "all"))
    return Routing(*_route(logits, int(k), bias, mask, normalize == "all"))


# ---------------------------------------------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------------------------------------------


def _loadable_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [R, C]`` as the tensor loads of the products take it: rows a multiple of 16 bytes apart, the first one aligned to
    16 bytes; ``t`` itself, or a copy with padded rows."""
    (ld, one), (r, c) = t.stride(), t.shape
    if one == 1 and ld >= c and ld % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    out = torch.empty((r, -(-c // 8) * 8), dtype=t.dtype, device=t.device)[:, :c]
    return out.copy_(t)


def _loadable_weights(w: torch.Tensor) -> torch.Tensor:
    """``w [E, N, K]`` itself where one of its two matrix dimensions is contiguous and the other strides are multiples of 16
    bytes, else a copy. Weights whose last dimension is a multiple of 8 are never copied."""
    e, n, k = w.shape
    se, sn, sk = w.stride()
    if w.data_ptr() % 16 == 0 and se % 8 == 0 and (se > 0 or e == 1):
        if sk == 1 and sn >= k and sn % 8 == 0 or sn == 1 and sk >= n and sk % 8 == 0:
            return w
    out = torch.empty((e, n, -(-k // 8) * 8), dtype=w.dtype, device=w.device)[:, :, :k]
    return out.copy_(w)


def _mm(x, rows, count, w, offsets, transposed=False, dtype=None):
    """``[count, N]``: rows of x (through ``rows``, if given) times their expert's matrix, or its transpose."""
    dev, (e, n, k), kind = x.device, w.shape, x.dtype
    x, w = _loadable_rows(x), _loadable_weights(w)
    se, sn, sk = w.stride()
    if transposed:
        n, k, sn, sk = k, n, sk, sn
    out = torch.empty((count, n), dtype=dtype or kind, device=dev)
    _lib.call("fs_grouped_mm", dev, x.data_ptr(), _ld(x), x.shape[0], _lib.ptr(rows), count, w.data_ptr(), se, sn, sk, e, n, k,
              offsets.data_ptr(), out.data_ptr(), _TYPES[dtype or kind], n, _TYPES[kind], _lib.stream_ptr(dev))
    return out


def _wgrad(dy, x, offsets):
    """``[E, N, K]``: per expert the sum over its rows of ``dy [R, N]`` times ``x [R, K]``."""
    dev, e, r = x.device, offsets.shape[0] - 1, x.shape[0]
    dy, x = _loadable_rows(dy), _loadable_rows(x)
    out = torch.empty((e, dy.shape[1], x.shape[1]), dtype=x.dtype, device=dev)
    _lib.call("fs_grouped_mm_wgrad", dev, _lib.ptr(dy), _ld(dy), _lib.ptr(x), _ld(x), r, e, dy.shape[1], x.shape[1],
              _lib.ptr(offsets), _lib.ptr(out), _TYPES[x.dtype], _lib.stream_ptr(dev))
    return out


def _gather(x, rows):
    """``x[rows]``, zeros for the rows of no pair."""
    return _combine(x, None, rows.view(-1, 1))


class _GroupedMmFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, rows, position, count):
        ctx.save_for_backward(x, w, offsets, rows, position)
        ctx.count = count
        return _mm(x, rows, count, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets, rows, position = ctx.saved_tensors
        dy = _loadable_rows(dy)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            if rows is None:
                dx = _mm(dy, None, ctx.count, w, offsets, transposed=True)
            else:  # rows in fp32, so that the sum over a token's rows is rounded once
                dx = _mm(dy, None, ctx.count, w, offsets, transposed=True, dtype=torch.float32)
                dx = _combine(dx, None, position, x.dtype)
        if ctx.needs_input_grad[1]:
            # a copy of the rows in order costs less than fetching them one by one for every tile of the product
            dw = _wgrad(dy, x if rows is None else _gather(x, rows), offsets)
        return dx, dw, None, None, None, None


def grouped_mm(x: torch.Tensor, weight: torch.Tensor, groups: Union[Routing, torch.Tensor], *,
               gather: bool = False) -> torch.Tensor:
    """``out[i] = weight[e] @ x[i]`` for the rows ``i`` of expert ``e``; zeros for the rows of no expert.

    ``groups``: a :class:`Routing`, or int32 offsets ``[E + 1]`` from 0 (group e has rows ``offsets[e]`` to
    ``offsets[e + 1]``; any sizes, zero among them). ``weight [E, N, K]`` as a linear layer holds it, or the transposed
    view of ``[E, K, N]``. ``x [R, K]`` in the order of the groups; with ``gather`` (and a routing) ``x [T, K]`` is in the
    order of the tokens and row ``i`` reads token ``routing.rows[i]``, without a copy. fp16 or bf16, both the same; sums in
    fp32, one rounding. Differentiable in both. Operands that tensor loads do not take (16 bytes of alignment, rows and
    experts a multiple of 8 values apart) are copied in every call: keep weights padded to a multiple of 8.
    """
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError(f"x must be 2D and weight 3D [E, N, K], got shapes {tuple(x.shape)} and {tuple(weight.shape)}")
    _check_type("x", x, (torch.float16, torch.bfloat16))
    if weight.dtype != x.dtype:
        raise ValueError(f"weight must be of the type of x ({x.dtype}), got {weight.dtype}")
    dev = _device_of("x", x, weight=weight)
    e, n, k = weight.shape
    if x.shape[1] != k or k == 0 or n == 0:
        raise ValueError(f"x must have as many columns as weight ({k} > 0), got {x.shape[1]}; N must be > 0, got {n}")
    rows = position = None
    if isinstance(groups, Routing):
        _check_routing(groups, dev, "offsets", *(("rows", "position") if gather else ()))
        offsets, (tokens, slots) = groups.offsets, groups.position.shape
        count = tokens * slots
        if gather:
            rows, position = groups.rows, groups.position
    else:
        if gather:
            raise ValueError("gather needs a Routing")
        _check_offsets(groups, dev)
        offsets, count = groups, x.shape[0]
    if x.shape[0] != (tokens if gather else count):
        raise ValueError(f"x must have {tokens if gather else count} rows, got {x.shape[0]}")
    if offsets.shape[0] != e + 1 or e > MAX_EXPERTS:
        raise ValueError(f"groups must have as many experts as weight ({e}, at most {MAX_EXPERTS}), got {offsets.shape[0] - 1}")
    x, weight = _loadable_rows(x), _loadable_weights(weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _GroupedMmFunction.apply(x, weight, offsets, rows, position, count)
    return _mm(x, rows, count, weight, offsets)


# ---------------------------------------------------------------------------------------------------------------
# Gated activation
# ---------------------------------------------------------------------------------------------------------------


def _act(u, gates, pairs, checkpoint):
    """The result, and with ``checkpoint`` one buffer with the codes ``[R, 2 F]`` and, behind them, their scales."""
    dev, (r, f2), kind = u.device, u.shape, u.dtype
    f = f2 // 2
    h = torch.empty((r, f), dtype=kind, device=dev)
    held = torch.empty(r * (f2 + 2 * (-(-f // _BLOCK))), dtype=torch.uint8, device=dev) if checkpoint else None
    codes = _lib.ptr(held)
    _lib.call("fs_gated_act", dev, u.data_ptr(), _TYPES[kind], _ld(u), r, f, _lib.ptr(gates), _lib.ptr(pairs), h.data_ptr(),
              codes, codes and codes + r * f2, _lib.stream_ptr(dev))
    return h, held


def _act_grad(u, held, gates, pairs, position, dh, want_gates, want_h):
    dev, (r, f), kind = dh.device, dh.shape, dh.dtype
    du = torch.empty((r, 2 * f), dtype=kind, device=dev)
    dgates = torch.empty_like(gates) if want_gates else None
    h = torch.empty((r, f), dtype=kind, device=dev) if want_h else None
    codes = _lib.ptr(held)
    _lib.call("fs_gated_act_grad", dev, _lib.ptr(u), 0 if u is None else _ld(u), codes, codes and codes + 2 * r * f, _TYPES[kind], r, f,
              _lib.ptr(gates), _lib.ptr(pairs), _lib.ptr(position), dh.data_ptr(), _ld(dh), du.data_ptr(), _lib.ptr(dgates),
              _lib.ptr(h), _lib.stream_ptr(dev))
    return du, dgates, h


class _GatedActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, gates, pairs, position, checkpoint):
        h, held = _act(u, gates, pairs, checkpoint)
        ctx.save_for_backward(None if checkpoint else u, held, gates, pairs, position)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        u, held, gates, pairs, position = ctx.saved_tensors
        du, dgates, _ = _act_grad(u, held, gates, pairs, position, _rows_of(dh), ctx.needs_input_grad[1], False)
        return du if ctx.needs_input_grad[0] else None, dgates, None, None, None


def gated_act(u: torch.Tensor, routing: Optional[Routing] = None, *, checkpoint: bool = True) -> torch.Tensor:
    """``silu(g) * v`` of ``u = [g | v]`` (``[R, 2 F]`` to ``[R, F]``), times the gate of each row's pair if a routing is given.

    Rows of no pair give zeros. Differentiable in ``u`` and ``routing.gates``. With ``checkpoint`` (the default) the backward
    pass works from ``u`` held in 8 bits, and ``u`` itself need not stay: blocks of 32 values along each half are held
    as integers times the smallest power of two at which the largest magnitude rounds to 127 at most, so a value is off by
    at most 1/128 of its block's largest (blocks with an infinity or NaN come back as NaN). ``checkpoint=False`` keeps
    ``u``. The result itself is of the unrounded ``u`` either way. fp32, fp16 or bf16.
    """
    if u.ndim != 2 or u.shape[1] == 0 or u.shape[1] % 2:
        raise ValueError(f"u must be 2D [R, 2 F] with F > 0, got shape {tuple(u.shape)}")
    _check_type("u", u)
    dev = _device_of("u", u)
    gates = pairs = position = None
    if routing is not None:
        _check_routing(routing, dev, "gates", "pairs", "position")
        gates, pairs, position = routing.gates, routing.pairs, routing.position
        if u.shape[0] != pairs.shape[0]:
            raise ValueError(f"u must have {pairs.shape[0]} rows, got {u.shape[0]}")
    u = _rows_of(u)
    if torch.is_grad_enabled() and (u.requires_grad or (gates is not None and gates.requires_grad)):
        return _GatedActFunction.apply(u, gates, pairs, position, bool(checkpoint))
    return _act(u, gates, pairs, False)[0]


# ---------------------------------------------------------------------------------------------------------------
# Back into tokens
# ---------------------------------------------------------------------------------------------------------------


def _combine(o, gates, position, dtype=None):
    dev, (t, k), (m, d), kind = o.device, position.shape, o.shape, o.dtype
    y = torch.empty((t, d), dtype=dtype or kind, device=dev)
    _lib.call("fs_combine", dev, o.data_ptr(), _TYPES[kind], _ld(o), m, t, k, d, _lib.ptr(gates), position.data_ptr(),
              y.data_ptr(), _TYPES[dtype or kind], _lib.stream_ptr(dev))
    return y


class _CombineFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, o, gates, position, pairs):
        keep = gates is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(o if keep else None, gates, position, pairs)
        ctx.width = o.shape[1]
        return _combine(o, gates, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        o, gates, position, pairs = ctx.saved_tensors
        dy, dev, (t, k) = _rows_of(dy), dy.device, position.shape
        do = torch.empty((t * k, ctx.width), dtype=dy.dtype, device=dev)
        dgates = torch.empty_like(gates) if o is not None else None
        _lib.call("fs_combine_grad", dev, _lib.ptr(o), _TYPES[dy.dtype], 0 if o is None else _ld(o), t, k, ctx.width,
                  _lib.ptr(gates), _lib.ptr(position), _lib.ptr(pairs), _lib.ptr(dy), _ld(dy), _lib.ptr(do),
                  _lib.ptr(dgates), _lib.stream_ptr(dev))
        return do if ctx.needs_input_grad[0] else None, dgates, None, None


def combine_rows(o: torch.Tensor, routing: Routing, *, weighted: bool = True) -> torch.Tensor:
    """Sums the experts' rows ``o [T * k, D]`` back into tokens: ``y[t] = sum_s gates[t, s] * o[position[t, s]]``.

    Slots without an expert add nothing; a token without any gets zeros. ``weighted=False`` leaves the gates out (they are in
    the rows already, as after :func:`gated_act` with a routing). Differentiable in ``o`` and ``routing.gates``; fp32, fp16
    or bf16, summed in fp32 in the order of the slots.
    """
    if o.ndim != 2 or o.shape[1] == 0:
        raise ValueError(f"o must be 2D [T * k, D] with D > 0, got shape {tuple(o.shape)}")
    _check_type("o", o)
    _check_routing(routing, _device_of("o", o), "gates", "pairs", "position")
    if o.shape[0] != routing.pairs.shape[0]:
        raise ValueError(f"o must have {routing.pairs.shape[0]} rows, got {o.shape[0]}")
    if routing.position.shape[1] > MAX_K:
        raise ValueError(f"k must be at most {MAX_K}, got {routing.position.shape[1]}")
    o, gates = _rows_of(o), routing.gates if weighted else None
    if torch.is_grad_enabled() and (o.requires_grad or (gates is not None and gates.requires_grad)):
        return _CombineFunction.apply(o, gates, routing.position, routing.pairs)
    return _combine(o, gates, routing.position)


# ---------------------------------------------------------------------------------------------------------------
# The layer
# ---------------------------------------------------------------------------------------------------------------


class _ExpertMlpFunction(torch.autograd.Function):
    """Keeps x, the routing and u (in 8 bits) from the forward pass. The gates are in the activation, so the backward pass
    needs neither the experts' outputs nor their gradients: both of its products with the outer weights read dy."""

    @staticmethod
    def forward(ctx, x, w_in, w_out, gates, offsets, pairs, rows, position, checkpoint):
        u = _mm(x, rows, pairs.shape[0], w_in, offsets)
        h, held = _act(u, gates, pairs, checkpoint)
        ctx.save_for_backward(x, w_in, w_out, gates, offsets, pairs, rows, position, None if checkpoint else u, held)
        return _combine(_mm(h, None, pairs.shape[0], w_out, offsets), None, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out, gates, offsets, pairs, rows, position, u, held = ctx.saved_tensors
        need_x, need_in, need_out, need_gates = ctx.needs_input_grad[:4]
        dy, count = _loadable_rows(dy), pairs.shape[0]
        dy = _gather(dy, rows)  # for two products
        dh = _mm(dy, None, count, w_out, offsets, transposed=True)
        du, dgates, h = _act_grad(u, held, gates, pairs, position, dh, need_gates, need_out)
        dx = _combine(_mm(du, None, count, w_in, offsets, transposed=True), None, position) if need_x else None
        dw_in = _wgrad(du, _gather(x, rows), offsets) if need_in else None
        dw_out = _wgrad(dy, h, offsets) if need_out else None
        return dx, dw_in, dw_out, dgates, None, None, None, None, None


def expert_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, routing: Routing, *,
               checkpoint: bool = True) -> torch.Tensor:
    """A layer of gated experts: ``y[t] = sum_s gates[t, s] * w_out[e] @ (silu(g) * v)``, ``[g | v] = w_in[e] @ x[t]``.

    ``x [T, D]``, ``w_in [E, 2 F, D]``, ``w_out [E, D, F]``, all fp16 or all bf16; differentiable in ``x``, the weights and
    ``routing.gates``. ``checkpoint`` as in :func:`gated_act`: of everything between x and y only the inner activations
    stay for the backward pass, in 8 bits, and the outer product's weight gradient uses the activation recomputed from
    them.
    """
    if x.ndim != 2 or w_in.ndim != 3 or w_out.ndim != 3:
        raise ValueError("x must be 2D, w_in and w_out 3D")
    _check_type("x", x, (torch.float16, torch.bfloat16))
    if w_in.dtype != x.dtype or w_out.dtype != x.dtype:
        raise ValueError(f"w_in and w_out must be of the type of x ({x.dtype}), got {w_in.dtype} and {w_out.dtype}")
    _check_routing(routing, _device_of("x", x, w_in=w_in, w_out=w_out), "gates", "offsets", "pairs", "rows", "position")
    (t, d), e, f = x.shape, w_in.shape[0], w_out.shape[2]
    if w_in.shape != (e, 2 * f, d) or w_out.shape != (e, d, f) or d == 0 or f == 0:
        raise ValueError(f"w_in must be [E, 2 F, {d}] and w_out [E, {d}, F], got {tuple(w_in.shape)} and {tuple(w_out.shape)}")
    if routing.position.shape[0] != t or routing.offsets.shape[0] != e + 1 or routing.position.shape[1] > MAX_K:
        raise ValueError(f"routing must be of {t} tokens and {e} experts, at most {MAX_K} for a token")
    x, w_in, w_out = _loadable_rows(x), _loadable_weights(w_in), _loadable_weights(w_out)
    r = routing
    if torch.is_grad_enabled() and any(v.requires_grad for v in (x, w_in, w_out, r.gates)):
        return _ExpertMlpFunction.apply(x, w_in, w_out, r.gates, r.offsets, r.pairs, r.rows, r.position, bool(checkpoint))
    u = _mm(x, r.rows, r.pairs.shape[0], w_in, r.offsets)
    h = _act(u, r.gates, r.pairs, False)[0]
    return _combine(_mm(h, None, r.pairs.shape[0], w_out, r.offsets), None, r.position)


def transport_bias(x: torch.Tensor, router: torch.Tensor, *, eps: float = 0.1, n_iters: int = 20,
                   load: Optional[torch.Tensor] = None, **solver_kwargs) -> torch.Tensor:
    """Prices ``[E]`` at which the experts' shares of the tokens are ``load`` (uniform by default), for :func:`route_tokens`.

    Solves the entropic transport from the tokens ``x [T, D]`` (uniform weights) to the rows of ``router [E, D]`` (weights
    ``load``, which sum to 1) with ``sinkhorn_flashstyle_alternating`` under the cost ``|x - w|^2 / 2``, and returns
    ``g_e + eps log load_e - |w_e|^2 / 2``: the plan's row of a token is largest where ``x.w_e`` plus that is. The result
    carries no gradient. ``eps`` is in the unit of the logits ``x.w``.
    """
    from flash_sinkhorn_b200.sinkhorn_solvers import sinkhorn_flashstyle_alternating

    if x.ndim != 2 or router.ndim != 2 or x.shape[1] != router.shape[1]:
        raise ValueError(f"x must be [T, D] and router [E, D], got {tuple(x.shape)} and {tuple(router.shape)}")
    if x.shape[0] == 0 or router.shape[0] == 0:
        raise ValueError("x and router must have rows")
    x, w = x.detach().float(), router.detach().float()
    (t, _), e = x.shape, w.shape[0]
    a = torch.full((t,), 1.0 / t, device=x.device)
    b = torch.full((e,), 1.0 / e, device=x.device) if load is None else load.detach().float()
    if b.shape != (e,):
        raise ValueError(f"load must have shape ({e},), got {tuple(b.shape)}")
    _, g = sinkhorn_flashstyle_alternating(x, w, a, b, eps=eps, n_iters=n_iters, cost_scale=0.5, **solver_kwargs)
    return g + eps * b.log() - 0.5 * (w * w).sum(1)
