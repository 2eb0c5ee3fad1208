"""The vocabulary's two ends: token embedding, and cross entropy over the vocabulary without its logits.

``token_embedding`` looks rows up and scales them; its
gradient adds the rows of every token in the order of its positions: positions are sorted
by id (a radix sort), sums run over sorted ranges in float32 without atomics, and tokens
that do not occur get their zeros in the same pass.  The same inputs give the same bits.

``linear_cross_entropy`` is the head and the loss of ``RavelLM.forward`` (``ravel_lm/model.py:506``) in one:

    z = x @ weight.T,   loss_i = log sum_v exp z_iv - z_i,target

The [rows, V] logits are never kept: a tensor-core kernel reduces each tile of them to
a maximum and a sum per row where they are made.  A training step makes the gradients of
a reduced loss in its forward, piece of rows by piece of rows: ``softmax - onehot`` in
16 bits (at most 512 MB or 1024 rows of it) from the logits' product done again -- large
bfloat16 steps get it from the first, as exp(z - z_target) and a factor per row -- and
its two products, in float32.  These float32 gradients (several slabs of one, where its product has few tiles) are held
until the graph goes; the backward scales them by the upstream gradient and rounds them once, so that it may be run again,
and a float16 loss scale loses nothing.  Single rows' losses (``reduction="none"``) get their
gradients in the backward, where the rows' upstream gradients are known.
Sums are float32.  What enters the gradients' products is rounded to 16 bits: the operands of either product, with
``reduction="none"`` the upstream gradient times ``softmax - onehot`` as a whole, in the three-product form (large
bfloat16 steps) exp(z - z_target) and, for the weight's gradient, x times the row's factor; the target's
own term, which carries most of a gradient, stays in float32 there.  In float16 what lies below 2^-40 of the
largest upstream gradient is dropped.

There is no CPU path, no float32 form of the cross entropy (parameters kept in float32, as under
autocast, are cast by the caller), no second derivative and no forward-mode one.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

Tensor = torch.Tensor

_REDUCTIONS = {"none": _lib.RAVEL_REDUCE_NONE, "sum": _lib.RAVEL_REDUCE_SUM, "mean": _lib.RAVEL_REDUCE_MEAN}


def token_embedding(ids: Tensor, weight: Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """``scale * weight[ids]``, differentiable in ``weight``.

    Args:
        ids:         [...] int32 or int64.  An id outside [0, V) gives zeros, has no gradient and sets
                     ``RAVEL_DEVERR_INDEX`` in the device error word.
        weight:      [V, K] float32, bfloat16 or float16; rows may be strided.
        padding_idx: the id whose positions give no gradient (negative: from the vocabulary's end).
    Returns:
        [..., K] of weight's dtype.
    """
    return _lib.host().token_embedding(ids, weight, float(scale), padding_idx)


def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Cross entropy of the logits ``x @ weight.T`` against ``targets``, differentiable in ``x`` and ``weight``.

    Args:
        x:            [..., K], bfloat16 or float16; rows may be strided.
        weight:       [V, K] of x's dtype.
        targets:      [...] int32 or int64.  Positions with ``ignore_index`` have loss 0 and gradient 0, whatever
                      their x holds.  Any other target outside [0, V) counts as ignored too and sets
                      ``RAVEL_DEVERR_INDEX`` in the device error word.
        reduction:    "mean" (over positions with a target; 0 without any), "sum" or "none".
    Returns:
        float32: a scalar, or [...] for "none".
    """
    try:
        code = _REDUCTIONS[reduction]
    except (KeyError, TypeError):
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, got {reduction!r}") from None
    return _lib.host().linear_cross_entropy(x, weight, targets, int(ignore_index), code)


__all__ = ["linear_cross_entropy", "token_embedding"]
