"""Tokens sorted by expert and back, with weights applied, and the gradients.

The projection layer can serve as a router: its output, a point of a polytope (a simplex
per token, a capacity per expert), holds the gates.  ``route_to_experts`` sorts the chosen
slots by expert, ``dispatch_to_experts`` puts each token's row where its experts read it,
``combine_from_experts`` adds the experts' rows up with the gates as weights; the gradient
with respect to the weights is the cotangent that the layer's implicit VJP takes.

Nothing is counted on the host: every slot has a sorted row, and slots without an expert
(a gate of zero) sort behind the last expert's rows.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from purin_b200 import _native_ops as _ops


class ExpertRouting(NamedTuple):
    """Slots sorted by expert (all int32, on the device).

    ``offsets[e]:offsets[e + 1]`` are expert e's sorted rows; ``position[t, k]`` is the
    sorted row of slot k of token t; ``source[r]`` is the slot ``t * slots + k`` of sorted
    row r.  Rows from ``offsets[-1]`` on belong to dropped slots.  A routing is used as
    ``route_to_experts`` made it, whole: a part of its tokens is routed anew.
    """

    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor

    @property
    def num_experts(self):
        return self.offsets.shape[0] - 1


def route_to_experts(experts, num_experts) -> ExpertRouting:
    """Sort the slots of ``experts`` (tokens, slots) by expert, stably.

    ``experts`` is int32 or int64; a value outside ``[0, num_experts)`` drops the slot.
    """
    what = "route_to_experts"
    _ops.require_cuda(what, experts)
    _ops.require_whole(what, "experts", experts)
    if experts.dim() != 2 or experts.shape[1] < 1:
        raise ValueError(f"{what}: experts must have shape (tokens, slots), got {tuple(experts.shape)}")
    num_experts = int(num_experts)
    if num_experts < 1:
        raise ValueError(f"{what}: num_experts must be positive")
    return ExpertRouting(*_ops.load().route(experts, num_experts))


def _check_routing(what, x, routing):
    """The routing is whole, and on the CUDA device of ``x``."""
    offsets, position, source = routing
    _ops.load().check_routing(what, x, offsets, position, source)


def _check_rows(what, name, t, rows):
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{what}: {name} must have shape ({rows}, dim), got {tuple(t.shape)}")
    _ops.require_floating(what, name, t)


def dispatch_to_experts(x, routing: ExpertRouting):
    """Rows of ``x`` (tokens, dim) in sorted order, (tokens * slots, dim); dropped rows are zero.

    Differentiable: a token's gradient is the sum of its kept slots' gradients.
    """
    what = "dispatch_to_experts"
    _check_routing(what, x, routing)
    _check_rows(what, "x", x, routing.position.shape[0])
    return _ops.load().dispatch(x, routing.offsets, routing.position)


def combine_from_experts(rows, weights, routing: ExpertRouting):
    """``out[t] = sum_k weights[t, k] * rows[position[t, k]]`` over the kept slots, (tokens, dim).

    ``rows`` is (tokens * slots, dim) in sorted order; ``weights`` (tokens, slots) in float32
    or float64.  Dropped slots' rows and weights are not read, whatever they hold, and get
    zero gradients; a token without a kept slot gives a zero row.  Sums are in 32 bits (64 for
    float64 rows).
    """
    what = "combine_from_experts"
    _check_routing(what, rows, routing)
    _ops.require_cuda(what, rows, weights)
    tokens, slots = routing.position.shape
    _check_rows(what, "rows", rows, tokens * slots)
    if weights.shape != (tokens, slots):
        raise ValueError(f"{what}: weights must have shape {(tokens, slots)}, got {tuple(weights.shape)}")
    if weights.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"{what}: weights must be float32 or float64, got {weights.dtype}")
    return _ops.load().combine(rows, weights, routing.offsets, routing.position)
