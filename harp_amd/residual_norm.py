"""The residual addition with its RMSNorm, on the GPU.

Every block of the model adds the attention's and the feed-forward's results
to the residual stream and normalises it before the next layer
(src/models/z_image/module/block.py).  :func:`add_rms_norm` is that pair in
one pass over the rows::

    h = x + residual                                # rounded to the residual's type
    y = h / sqrt(mean(h^2) + eps) * weight          # in x's type

and differentiable (:class:`AddRMSNormFn`: one kernel for the gradients of x
and the residual, one small reduction for the weight's).
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

from . import _lib
from .int8 import Int8Rows, _refuse_grad


def _ops():
    _lib.load_block_ops()
    return torch.ops.harp_block


class AddRMSNormFn(torch.autograd.Function):
    """(y, h) of (x, residual, weight, eps); y alone where residual is None."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _ops().add_rms_norm_forward(x, residual, weight, eps, True)
        ctx.set_materialize_grads(False)
        ctx.x_dtype = x.dtype
        if residual is None:
            ctx.save_for_backward(x, weight, rstd)
            return y
        ctx.save_for_backward(h, weight, rstd)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # y took no part: the addition alone
            return (dh.to(ctx.x_dtype) if need_x and dh is not None else None), (dh if need_res else None), None, None
        dx, dres, gw = _ops().add_rms_norm_backward(dy, dh, h, weight, rstd, need_res, need_w)
        if need_res and dres.numel() == 0:
            dres = dx  # the same values in the same type
        return dx if need_x else None, dres if need_res else None, gw if need_w else None, None


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual in the residual's type (x itself without a
    residual), y = h / sqrt(mean(h^2) + eps) * weight in x's type."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        if residual is None:
            return AddRMSNormFn.apply(x, None, weight, float(eps)), x
        return AddRMSNormFn.apply(x, residual, weight, float(eps))
    y, h, _ = _ops().add_rms_norm_forward(x, residual, weight, float(eps), False)
    return y, (x if residual is None else h)


def add_rms_norm_int8(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Tuple[Int8Rows, torch.Tensor]:
    """(rows, h): as :func:`add_rms_norm` with y as 8-bit rows, quantised from
    float32.  Forward only: raises where a gradient would be recorded."""
    _refuse_grad("add_rms_norm_int8", x, residual, weight)
    values, scales, h = _ops().add_rms_norm_int8(x, residual, weight, float(eps))
    return Int8Rows(values, scales), (x if residual is None else h)
