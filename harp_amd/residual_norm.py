"""The residual addition with its RMSNorm, on the GPU.

The model's blocks add the attention's and the feed-forward's results to the
residual stream and normalise it before the next layer
(src/models/z_image/module/block.py).  :func:`add_rms_norm` is that pair in
one pass over the rows::

    h = x + residual                                # rounded to the residual's type
    y = h / sqrt(mean(h^2) + eps) * weight          # in x's type

and differentiable, once and in reverse mode (one kernel for the gradients of x
and the residual, one small reduction for the weight's).  There is no factor per
sample on the norm's result and no gate on the addition: a block with such a
modulation multiplies x before the call, and y after it.
:func:`add_rms_norm_int8` gives y as 8-bit rows instead
(:class:`harp_amd.Int8Rows`), for a Linear layer in 8-bit integers; it is
forward only.

x and the residual are bfloat16 or float32, each its own, of any matching
shape [.., C] with C up to 32768; the weight is a bfloat16 or float32 [C]
vector or None.  Statistics and sums are float32.  There is no CPU path.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .int8 import Int8Rows, _ops, _refuse_grad


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual in the residual's type (x itself without a
    residual), y = h / sqrt(mean(h^2) + eps) * weight in x's type."""
    y, h = _ops().add_rms_norm(x, residual, weight, eps)
    return y, (x if residual is None else h)


def add_rms_norm_int8(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Tuple[Int8Rows, torch.Tensor]:
    """(rows, h): as :func:`add_rms_norm` with y as 8-bit rows, quantised from
    float32.  Forward only: raises where a gradient would be recorded."""
    _refuse_grad("add_rms_norm_int8", x, residual, weight)
    values, scales, h = _ops().add_rms_norm_int8(x, residual, weight, eps)
    return Int8Rows(values, scales), (x if residual is None else h)
