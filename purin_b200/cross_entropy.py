"""Linear layer and softmax cross entropy over a vocabulary, without keeping the logits.

``linear_cross_entropy`` is the loss of a model whose states are trained through the
projection layer: ``z = hidden @ weight.T`` is made in pieces, reduced to its
log-sum-exp and the target's logit, and made again piece by piece for the gradients.
"""

from __future__ import annotations

import torch

from purin_b200 import _native_ops as _ops

_WHAT = "linear_cross_entropy"
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(hidden, weight, targets, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` against ``targets``, in float32.

    ``hidden`` (tokens, dim) and ``weight`` (vocab, dim) are bfloat16 or float32, of one
    type; ``targets`` (tokens) int32 or int64.  A target equal to ``ignore_index`` or outside
    ``[0, vocab)`` gives no loss and no gradient.  ``reduction`` is "mean" (over the targets
    that count; 0 if none does), "sum" or "none".  Differentiable in ``hidden`` and ``weight``;
    the logits are not kept, the backward makes them again.  bfloat16 products are exact and
    summed in float32 by an adder that truncates (a mean loss is off by some 5e-7 of itself), and the
    logits' gradient is rounded to bfloat16 before its products.  float32 operands keep float32
    accuracy, and have to be finite: the parts of an infinite one can make its logits NaN.
    Beside its outputs a backward holds 256 MB of the logits' gradient at most, or 1024 columns of it
    where those are more (2 bytes a value for bfloat16, 6 for float32).  Should a kernel's bounded
    wait run out, every loss or gradient of the call is NaN.
    """
    _ops.require_cuda(_WHAT, hidden, weight, targets)
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1] \
            or hidden.shape[1] < 1 or weight.shape[0] < 1:
        raise ValueError(f"{_WHAT}: hidden must be (tokens, dim) and weight (vocab, dim), got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{_WHAT}: hidden and weight must both be bfloat16 or float32, got "
                        f"{hidden.dtype} and {weight.dtype}")
    if targets.shape != hidden.shape[:1]:
        raise ValueError(f"{_WHAT}: targets must have shape {tuple(hidden.shape[:1])}, got "
                         f"{tuple(targets.shape)}")
    _ops.require_whole(_WHAT, "targets", targets)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{_WHAT}: reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    return _ops.load().linear_cross_entropy(hidden, weight, targets, int(ignore_index),
                                            _REDUCTIONS[reduction])
