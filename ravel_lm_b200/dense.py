"""A Linear with its epilogue on the 5th-generation tensor cores.

The projections of a RAVEL layer around the memory -- the packed input GEMM
(``ravel_lm/model.py:329``), the ``fuse`` read-out with its residual (``:386``),
the feed-forward products, the head -- are Linears followed by elementwise work.
``fused_linear`` computes

    y = residual + activation(x @ weight.T + bias)

in one kernel for bfloat16 or float16 tensors: products accumulated in float32
in tensor memory, bias, activation and residual applied there, one rounding.
Training saves x, the weight and (with an activation) the sum before it in 16
bits; the backward makes ``dz = dy * activation'(z)`` together with the bias
gradient in one pass, then the two gradient products on the same tensor-core
kernel, which reads each operand as it lies.  Calls with few rows (decoding)
divide the contraction over a cluster of CTAs.

Leading dimensions are arbitrary and may be strided or empty.  Rows that TMA
cannot read in place (a pitch or an address that is no multiple of 16 bytes)
are copied once to a padded pitch.  Every result is deterministic.  There is no
CPU path, no float32 form (parameters kept in float32, as under autocast, are cast by
the caller), no second derivative (``create_graph`` is refused) and no forward-mode
one (tangents are refused).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

Tensor = torch.Tensor

_ACTIVATIONS = {"none": _lib.RAVEL_ACT_NONE, "relu": _lib.RAVEL_ACT_RELU, "gelu": _lib.RAVEL_ACT_GELU,
                "silu": _lib.RAVEL_ACT_SILU}


def fused_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: str = "none",
                 residual: Optional[Tensor] = None) -> Tensor:
    """``residual + activation(x @ weight.T + bias)``, differentiable in every tensor.

    Args:
        x:          [..., K], bfloat16 or float16.
        weight:     [N, K] of x's dtype (``torch.nn.Linear.weight``).
        bias:       optional [N].
        activation: "none", "relu", "gelu" (z * Phi(z), with the error function) or "silu".
        residual:   optional [..., N], added after the activation.
    Returns:
        [..., N] of x's dtype.
    """
    try:
        act = _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}") from None
    return _lib.host().fused_linear(x, weight, bias, residual, act)


__all__ = ["fused_linear"]
