"""Distillation from a teacher's top logits, forward and backward.

A RAVEL model that learns from a larger one is trained on the teacher's k largest
logits per position (stored with the corpus; whole rows would be far too large).
With temperature T, p = softmax(teacher / T) over a position's entries and
q = softmax(logits / T) over the vocabulary, a position's loss is

    T^2 sum_j p_j (log p_j - log q[id_j])

(the factor T^2 keeps the gradient's scale independent of T).  Entries with a
negative id (padding of ragged lists) or a teacher logit of -inf do not exist; a
position without any entry has loss 0, gradient 0 and is not counted by the mean.
Entries that name the same id add up.

The student's logits are read once: a running maximum and sum per row.  In a
training step the same kernel writes the gradient while the row is still in L2,
for an upstream gradient of 1 (``loss.backward()``; ``weight`` scales the loss where
it is one term of several, so that its upstream gradient stays 1); with any other
upstream gradient the backward computes it from the logits again, as it does for
float16 logits and for ``reduction="none"``.  The gradient's memory is thus held from
the forward on, until the backward takes it or the graph goes; saved-tensor hooks do not see it.
The search for entries of the same id costs k^2 a row: some hundreds of entries are cheap, thousands
take longer than the logits.  Sums are float32, of exponentials of differences from the row's
largest logit; results are deterministic.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib

Tensor = torch.Tensor

_REDUCTIONS = {"none": _lib.RAVEL_REDUCE_NONE, "sum": _lib.RAVEL_REDUCE_SUM, "mean": _lib.RAVEL_REDUCE_MEAN}


def distill_topk_loss(logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, *, temperature: float = 1.0,
                      reduction: str = "mean", weight: float = 1.0) -> Tensor:
    """``weight * T^2 KL(teacher's top k || student)`` per position, reduced; differentiable in ``logits``.

    Args:
        logits:         [..., V] float32, bfloat16 or float16; rows may be strided.
        teacher_ids:    [..., k] int32 or int64, k <= 4096; a negative id is an empty entry.  An id of V or
                        more is not used either and sets ``RAVEL_DEVERR_INDEX`` in the device error word.
        teacher_logits: [..., k] float32, bfloat16 or float16, without gradient.
        reduction:      "mean" (over positions that have an entry), "sum" or "none".
    Returns:
        float32: a scalar, or [...] for "none".
    """
    try:
        code = _REDUCTIONS[reduction]
    except (KeyError, TypeError):
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, got {reduction!r}") from None
    return _lib.host().distill_topk_loss(logits, teacher_ids, teacher_logits, float(temperature), float(weight), code)


__all__ = ["distill_topk_loss"]
