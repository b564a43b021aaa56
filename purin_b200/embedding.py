"""Embedding lookup with scaling; the table's gradient by sorted tokens.

``token_embedding`` turns token ids into the rows that a network feeds the projection
layer with.  Its gradient sorts the tokens by id and sums each id's rows in the tokens'
order, in 32 bits (64 for float64), so it is the same from run to run.
"""

from __future__ import annotations

import torch

from purin_b200 import _native_ops as _ops

_WHAT = "token_embedding"


def token_embedding(table, ids, *, scale=1.0, padding_index=None):
    """``scale * table[ids]``, of shape ``ids.shape + (dim,)``; differentiable in ``table``.

    ``table`` is (vocab, dim) in float64, float32, bfloat16 or float16 (rows may be strided);
    ``ids`` int32 or int64 of any shape.  An id outside ``[0, vocab)``, or equal to
    ``padding_index``, gives a zero row and no gradient: ids are not checked on the host.
    """
    _ops.require_cuda(_WHAT, table, ids)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"{_WHAT}: table must have shape (vocab, dim), got {tuple(table.shape)}")
    _ops.require_floating(_WHAT, "table", table)
    _ops.require_whole(_WHAT, "ids", ids)
    if padding_index is not None and not 0 <= int(padding_index) < table.shape[0]:
        raise ValueError(f"{_WHAT}: padding_index must be a row of the table")
    if isinstance(scale, torch.Tensor) and scale.requires_grad and torch.is_grad_enabled():
        raise TypeError(f"{_WHAT}: scale must be a number, got a tensor that needs a gradient")
    return _ops.load().embedding(table, ids, float(scale),
                                 -1 if padding_index is None else int(padding_index))
