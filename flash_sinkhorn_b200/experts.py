"""Routed experts, balanced by entropic transport: the operators between a router and its tokens.

Tokens and the rows of a router are two clouds, and a plan between them with uniform marginals sends the same share of
tokens to every expert. Since ``|x - w|^2 / 2 = |x|^2 / 2 + |w|^2 / 2 - x.w``, the plan of the framework's solver is
largest where ``x.w_e + bias_e`` is, with one price per expert: :func:`transport_bias`. What uses the prices is here:

* :func:`route_tokens` - the k experts of every token, their gates, and the order of the rows (:class:`Routing`);
* :func:`grouped_mm` - the experts' matrix products over groups of any size, one row or thousands;
* :func:`gated_act` - ``gate * silu(g) * v``, with its input kept in 8 bits for the backward pass;
* :func:`combine_rows` - the experts' rows summed back into tokens;
* :func:`expert_mlp` - the three in a row, as one layer with one backward pass.

And what stands around such a layer:

* :func:`layer_norm` - the norm in front of the router and the experts;
* :func:`grouped_mm8` - the experts' products in 8-bit floating point, with weights held so (:class:`Blocks8`,
  :func:`to_blocks8`) or put into 8 bits in every step; :func:`expert_mlp` takes held weights too;
* :func:`orthogonalize` - the update of the experts' matrices with all singular values brought to about 1.

All of it runs on the current stream of the tensors' device, never waits for the host (group sizes stay on the device, so
a call can be captured in a CUDA graph), and gives the same bits in every run. Sums are held in fp32. Waits inside the
products are bounded: should one ever give up, the results it leaves are NaN and the library's health word is set
(``fs_device_error()``, which waits for the device). Extension without a
counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from flash_sinkhorn_b200 import _lib

__all__ = ["Routing", "Blocks8", "route_tokens", "grouped_mm", "grouped_mm8", "to_blocks8", "gated_act", "combine_rows", "expert_mlp",
           "layer_norm", "orthogonalize", "transport_bias"]


class Routing(NamedTuple):
    """Where the rows of ``T`` tokens and ``k`` slots go; row ``i`` of a grouped tensor belongs to pair ``pairs[i]``."""

    gates: torch.Tensor  #: ``[T, k]`` float32, 0 for a slot without an expert; differentiable
    experts: torch.Tensor  #: ``[T, k]`` int32, -1 for a slot without an expert
    offsets: torch.Tensor  #: ``[E + 1]`` int32; expert e has rows ``offsets[e]`` to ``offsets[e + 1]``
    pairs: torch.Tensor  #: ``[T * k]`` int32 pair (``token * k + slot``) of each row, -1 after the last routed one
    rows: torch.Tensor  #: ``[T * k]`` int32 token of each row, -1 after the last routed one
    position: torch.Tensor  #: ``[T, k]`` int32 row of each pair, -1 for a slot without an expert


class Blocks8(NamedTuple):
    """Weights ``[E, N, K]`` in 8-bit floating point, a scale for each block of 128 x 128: ``codes * scales`` stands for them.

    What :func:`to_blocks8` gives, or codes and scales from elsewhere: scales may have any finite value, not powers of two only.
    """

    codes: torch.Tensor  #: ``[E, N, K]`` float8_e4m3fn; rows a multiple of 16 values apart, or every call copies them
    scales: torch.Tensor  #: ``[E, ceil(N / 128), ceil(K / 128)]`` float32


def _check_routing(routing) -> None:
    if not isinstance(routing, Routing):
        raise ValueError(f"routing must be a Routing, got {type(routing).__name__}")


def route_tokens(logits: torch.Tensor, k: int, *, bias: Optional[torch.Tensor] = None,
                 mask: Optional[torch.Tensor] = None, normalize: str = "selected") -> Routing:
    """Chooses ``k`` experts for every row of ``logits [T, E]`` and puts the pairs in the order of the experts.

    The chosen ones have the largest ``logits + bias`` (in fp32; ties go to the lower expert, NaN comes first so that it
    shows in the gates); ``bias [E]``, for instance prices of :func:`transport_bias`, only takes part in the choice.
    Experts whose logit or bias is ``-inf``, and all experts of tokens whose ``mask [T]`` is False, are never chosen. Gates
    are the soft-max of the logits over the chosen experts (``normalize="selected"``) or over all experts that can be
    chosen (``"all"``), and carry the gradient to ``logits`` (fp32, fp16 or bf16). At most 1024 experts and 32 slots.
    """
    if normalize not in ("selected", "all"):
        raise ValueError(f"normalize must be 'selected' or 'all', got {normalize!r}")
    return Routing(*_lib.torch_binding().route_tokens(logits, int(k), bias, mask, normalize == "all"))


def grouped_mm(x: torch.Tensor, weight: torch.Tensor, groups: Union[Routing, torch.Tensor], *,
               gather: bool = False) -> torch.Tensor:
    """``out[i] = weight[e] @ x[i]`` for the rows ``i`` of expert ``e``; zeros for the rows of no expert.

    ``groups``: a :class:`Routing`, or int32 offsets ``[E + 1]`` from 0 (group e has rows ``offsets[e]`` to
    ``offsets[e + 1]``; any sizes, zero among them). ``weight [E, N, K]`` as a linear layer holds it, or the transposed
    view of ``[E, K, N]``. ``x [R, K]`` in the order of the groups; with ``gather`` (and a routing) ``x [T, K]`` is in the
    order of the tokens and row ``i`` reads token ``routing.rows[i]``; batches of thousands of rows are copied into order
    first, ``R * K`` values that live for the call. fp16 or bf16, both the same; sums in fp32, one rounding. Differentiable in both. Operands that tensor loads do not take (16 bytes of alignment, rows and
    experts a multiple of 8 values apart) are copied in every call: keep weights padded to a multiple of 8.
    """
    if isinstance(groups, Routing):
        return _lib.torch_binding().grouped_mm(x, weight, groups.offsets, groups.rows, groups.position, bool(gather))
    if gather:
        raise ValueError("gather needs a Routing")
    return _lib.torch_binding().grouped_mm(x, weight, groups, None, None, False)


def to_blocks8(weight: torch.Tensor) -> Blocks8:
    """``weight [E, N, K]`` (fp16 or bf16) in 8 bits, for :func:`grouped_mm8` and :func:`expert_mlp`. Carries no gradient.

    The scale of 128 x 128 values is the smallest power of two (from ``2**-126`` on) at which their largest magnitude is at most 448,
    and each value is rounded to the nearest code, ties to even: off by at most 1/16 of itself, or ``2**-10`` of the scale if
    that is more. A block with an infinity or a NaN has the scale NaN, and the products that read it are NaN.
    """
    return Blocks8(*_lib.torch_binding().to_blocks8(weight))


def grouped_mm8(x: torch.Tensor, weight: Union[Blocks8, torch.Tensor], groups: Union[Routing, torch.Tensor], *,
                gather: bool = False) -> torch.Tensor:
    """:func:`grouped_mm` in 8-bit floating point: ``out[i] = q(weight[e]) @ q(x[i])``, in the type of x (fp16 or bf16).

    ``x`` is put into 8 bits in every call, blocks of 128 values along its rows with a scale each, as :func:`to_blocks8` does
    blocks of 128 x 128; so is ``weight`` given as a tensor ``[E, N, K]`` of the type of x (training). A :class:`Blocks8` is taken as it
    is (serving). ``groups`` and ``gather`` as in :func:`grouped_mm`. Sums are fp32, within blocks of 128 by the tensor core; one rounding.

    Differentiable in x and in a ``weight`` given as a tensor: the roundings to 8 bits count as the identity. The gradient to x is
    ``q(dy) @ q(weight[e])``, with blocks of 128 along the rows of ``dy`` and the same codes of the weights; that to ``weight`` is
    the 16-bit product of ``dy`` and ``x`` as they are.
    """
    held = isinstance(weight, Blocks8)
    w, codes, scales = (None, *weight) if held else (weight, None, None)
    if isinstance(groups, Routing):
        return _lib.torch_binding().grouped_mm8(x, w, codes, scales, groups.offsets, groups.rows, groups.position, bool(gather))
    if gather:
        raise ValueError("gather needs a Routing")
    return _lib.torch_binding().grouped_mm8(x, w, codes, scales, groups, None, None, False)


def gated_act(u: torch.Tensor, routing: Optional[Routing] = None, *, checkpoint: bool = True) -> torch.Tensor:
    """``silu(g) * v`` of ``u = [g | v]`` (``[R, 2 F]`` to ``[R, F]``), times the gate of each row's pair if a routing is given.

    Rows of no pair give zeros. Differentiable in ``u`` and ``routing.gates``. With ``checkpoint`` (the default) the backward
    pass works from ``u`` held in 8 bits, and ``u`` itself need not stay: blocks of 32 values along each half are held
    as integers times the smallest power of two at which the largest magnitude rounds to 127 at most, so a value is off by
    at most 1/127.5 of its block's largest (blocks with an infinity or NaN come back as NaN). ``checkpoint=False`` keeps
    ``u``, and the gradients are those of the unrounded values (with the checkpoint they are off by a percent or so, the price of
    half the memory). The result itself is of the unrounded ``u`` either way. fp32, fp16 or bf16; the sigmoid to a relative
    ``2**-21``, for ``g`` below 0 ``|g| * 2**-23`` more, and 0 for ``g`` below -87.3.
    """
    if routing is None:
        return _lib.torch_binding().gated_act(u, None, None, None, bool(checkpoint))
    _check_routing(routing)
    return _lib.torch_binding().gated_act(u, routing.gates, routing.pairs, routing.position, bool(checkpoint))


def combine_rows(o: torch.Tensor, routing: Routing, *, weighted: bool = True) -> torch.Tensor:
    """Sums the experts' rows ``o [T * k, D]`` back into tokens: ``y[t] = sum_s gates[t, s] * o[position[t, s]]``.

    Slots without an expert add nothing; a token without any gets zeros. ``weighted=False`` leaves the gates out (they are in
    the rows already, as after :func:`gated_act` with a routing). Differentiable in ``o`` and ``routing.gates``; fp32, fp16
    or bf16, summed in fp32 in the order of the slots.
    """
    _check_routing(routing)
    return _lib.torch_binding().combine_rows(o, routing.gates, routing.pairs, routing.position, bool(weighted))


def expert_mlp(x: torch.Tensor, w_in: Union[torch.Tensor, Blocks8], w_out: Union[torch.Tensor, Blocks8], routing: Routing, *,
               checkpoint: bool = True) -> torch.Tensor:
    """A layer of gated experts: ``y[t] = sum_s gates[t, s] * w_out[e] @ (silu(g) * v)``, ``[g | v] = w_in[e] @ x[t]``.

    ``x [T, D]``, ``w_in [E, 2 F, D]``, ``w_out [E, D, F]``, all fp16 or all bf16; differentiable in ``x``, the weights and
    ``routing.gates``. ``checkpoint`` as in :func:`gated_act`: of everything between x and y only the inner activations
    stay for the backward pass, in 8 bits, and the outer product's weight gradient uses the activation recomputed from
    them. The operators' results between x and y are of the type of x (a token's rows of the second product are rounded,
    then summed in fp32 and rounded again), as are the gradients between dy and dx, but for the rows that are summed to
    dx, which are fp32.

    With both weights given as :class:`Blocks8` the products are those of :func:`grouped_mm8`; differentiable in ``x`` and
    ``routing.gates`` then.
    """
    _check_routing(routing)
    if isinstance(w_in, Blocks8) or isinstance(w_out, Blocks8):
        if not (isinstance(w_in, Blocks8) and isinstance(w_out, Blocks8)):
            raise ValueError("w_in and w_out must both be Blocks8, or neither")
        n_in, n_out = w_in.codes.shape, w_out.codes.shape
        if x.ndim != 2 or len(n_in) != 3 or n_in[1:] != (2 * n_out[-1], x.shape[1]) or n_out[:-1] != (n_in[0], x.shape[1]):
            raise ValueError(f"x must be [T, D], w_in [E, 2 F, D] and w_out [E, D, F], got {tuple(x.shape)}, {tuple(n_in)} and {tuple(n_out)}")
        h = gated_act(grouped_mm8(x, w_in, routing, gather=True), routing, checkpoint=checkpoint)
        return combine_rows(grouped_mm8(h, w_out, routing), routing, weighted=False)
    r = routing
    return _lib.torch_binding().expert_mlp(x, w_in, w_out, r.gates, r.offsets, r.pairs, r.rows, r.position, bool(checkpoint))


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x [..., F]`` (fp32, fp16 or bf16), in its type.

    ``weight`` and ``bias`` ``[F]``: float32 or the type of x, both the same; either may be left out. Differentiable in all three;
    mean and deviation stay for the backward pass, and the sums over the rows for ``weight`` and ``bias`` are fp32 in a fixed order.
    """
    return _lib.torch_binding().layer_norm(x, weight, bias, float(eps))


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Brings the singular values of each matrix of ``g [..., N, K]`` to about 1 and leaves its singular vectors, for updates.

    ``X = g / (|g| + eps)`` with the Frobenius norm, then ``steps`` times ``X <- a X + b (X X^T) X + c (X X^T)^2 X`` with
    ``coefficients = (a, b, c)``; the default ones bring values from 0.003 on to between 0.68 and 1.21 in five steps. ``g`` is fp32, fp16 or
    bf16, the result of ``dtype`` (fp16 or bf16) and carries no gradient. Products are of fp16 operands with fp32 sums, the part
    ``a X`` is of 22 bits in all steps but the last: the result is off by 0.05 to 0.3 % of its norm besides its rounding. Roundings of few entries do
    not average: with 16 rows or columns it may be 0.5 %, with one to four 1 % and in rare cases 2 to 3 %. Coefficients have to keep the
    singular values at 2 or less. A matrix with an infinity or a NaN gives NaN, zeros give zeros.
    """
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
    a, b, c = (float(v) for v in coefficients)
    return _lib.torch_binding().orthogonalize(g, int(steps), a, b, c, float(eps), dtype == torch.bfloat16)


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
