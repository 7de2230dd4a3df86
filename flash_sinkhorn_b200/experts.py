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
a call can be captured in a CUDA graph), and gives the same bits in every run. Sums are held in fp32. Waits inside the
products are bounded: should one ever give up, the results it leaves are NaN and the library's health word is set
(``fs_device_error()``, which waits for the device). Extension without a
counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from flash_sinkhorn_b200 import _lib

__all__ = ["Routing", "route_tokens", "grouped_mm", "gated_act", "combine_rows", "expert_mlp", "transport_bias"]


class Routing(NamedTuple):
    """Where the rows of ``T`` tokens and ``k`` slots go; row ``i`` of a grouped tensor belongs to pair ``pairs[i]``."""

    gates: torch.Tensor  #: ``[T, k]`` float32, 0 for a slot without an expert; differentiable
    experts: torch.Tensor  #: ``[T, k]`` int32, -1 for a slot without an expert
    offsets: torch.Tensor  #: ``[E + 1]`` int32; expert e has rows ``offsets[e]`` to ``offsets[e + 1]``
    pairs: torch.Tensor  #: ``[T * k]`` int32 pair (``token * k + slot``) of each row, -1 after the last routed one
    rows: torch.Tensor  #: ``[T * k]`` int32 token of each row, -1 after the last routed one
    position: torch.Tensor  #: ``[T, k]`` int32 row of each pair, -1 for a slot without an expert


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


def expert_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, routing: Routing, *,
               checkpoint: bool = True) -> torch.Tensor:
    """A layer of gated experts: ``y[t] = sum_s gates[t, s] * w_out[e] @ (silu(g) * v)``, ``[g | v] = w_in[e] @ x[t]``.

    ``x [T, D]``, ``w_in [E, 2 F, D]``, ``w_out [E, D, F]``, all fp16 or all bf16; differentiable in ``x``, the weights and
    ``routing.gates``. ``checkpoint`` as in :func:`gated_act`: of everything between x and y only the inner activations
    stay for the backward pass, in 8 bits, and the outer product's weight gradient uses the activation recomputed from
    them. The operators' results between x and y are of the type of x (a token's rows of the second product are rounded,
    then summed in fp32 and rounded again), as are the gradients between dy and dx, but for the rows that are summed to
    dx, which are fp32.
    """
    _check_routing(routing)
    r = routing
    return _lib.torch_binding().expert_mlp(x, w_in, w_out, r.gates, r.offsets, r.pairs, r.rows, r.position, bool(checkpoint))


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
