"""Rotary positions with several axes, on the GPU.

A token of an image or a video has a position along each of a few axes (time,
height, width; the model's RopeEmbedder, src/models/z_image/
standalone_transformer.py).  Each axis turns its own share of a head's feature
pairs: pair j of an axis of ``width`` features turns by
``position * theta ** (-2 j / width)`` radians.

:class:`AxialRope` describes the axes.  :func:`qk_norm_axial_rope` normalises
queries and keys over each head's features and rotates them by their tokens'
positions, both in one pass over memory and differentiable;
:meth:`AxialRope.table` gives the complex table that the operators which take
``freqs_cis`` read.  :class:`AxialPositions` stands in the place of that table
for :func:`harp_amd.project_qkv` and :class:`harp_amd.RingZAttention`.

Angles are formed in 64 bits, so far positions keep their precision; the rest is
32-bit arithmetic over bfloat16 or float32 tensors, rounded once, to nearest.
There is no CPU path.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib

MAX_AXES = _lib.HARP_REQ_MAX_AXES

_harp_request = None


def _ops():
    """torch.ops.harp_request, its library loaded at the first call."""
    global _harp_request
    if _harp_request is None:
        _lib.load_request_ops()
        _harp_request = torch.ops.harp_request
    return _harp_request


class AxialRope:
    """The axes of a rotary embedding, for heads of ``sum(axes_dims)`` features.

    ``axes_dims``: how many features each of one to four axes turns (even), in the
    order of a head's pairs; ``theta``: one base for all axes or one for each;
    ``layout``: pairs are neighbours (2p, 2p + 1), ``"interleaved"``, as the
    model's complex tables have them, or (p, p + D / 2), ``"half"``."""

    __slots__ = ("axes_dims", "theta", "layout")

    def __init__(self, axes_dims: Sequence[int], theta: Union[float, Sequence[float]],
                 layout: str = "interleaved"):
        self.axes_dims = tuple(int(d) for d in axes_dims)
        thetas = (theta,) * len(self.axes_dims) if isinstance(theta, (int, float)) else tuple(theta)
        self.theta = tuple(float(t) for t in thetas)
        self.layout = layout
        if not 1 <= len(self.axes_dims) <= MAX_AXES or any(d < 2 or d % 2 for d in self.axes_dims):
            raise ValueError(f"axes_dims must be one to {MAX_AXES} even widths, got {tuple(axes_dims)}")
        if len(self.theta) != len(self.axes_dims) or any(not (t > 0 and math.isfinite(t)) for t in self.theta):
            raise ValueError(f"theta must be a positive number, or one for each of {len(self.axes_dims)} axes, got {theta}")
        if layout not in ("interleaved", "half"):
            raise ValueError(f'layout must be "interleaved" or "half", got {layout!r}')

    @property
    def dim(self) -> int:
        """Features of a head."""
        return sum(self.axes_dims)

    def table(self, positions: torch.Tensor) -> torch.Tensor:
        """exp(i angle) of every pair, complex64 [.., S, D / 2], of positions [S, axes] or [B, S, axes]."""
        return _ops().rope_table(positions, self.axes_dims, self.theta)

    def __repr__(self) -> str:
        return f"AxialRope(axes_dims={self.axes_dims}, theta={self.theta}, layout={self.layout!r})"


class AxialPositions(NamedTuple):
    """Tokens' positions [S, axes] or [B, S, axes] (int32, int64 or float32), and the axes they are along."""

    positions: torch.Tensor
    rope: AxialRope

    def table(self) -> torch.Tensor:
        """The complex table of these positions (:meth:`AxialRope.table`)."""
        return self.rope.table(self.positions)


_Eps = Union[None, float, Tuple[Optional[float], Optional[float]]]


def qk_norm_axial_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: AxialRope,
                       q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                       eps: _Eps = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q, k), each head normalised (where ``eps`` is given) and rotated by its token's positions.

    q and k: bfloat16 or float32 [B, heads, S, D], each with heads of its own number and any
    strides; k may be None.  ``positions``: [S, axes] for all of the batch, or [B, S, axes].
    ``eps``: of the RMSNorms in front of the rotation, one number or one for q and one for k; None
    leaves the norm out.  The weights are bfloat16 or float32 [D] vectors, or None for a norm without one.
    The results have q's and k's layouts, without the holes these may have (features are neighbours
    always).  Gradients of q, k and the weights, once and in reverse mode."""
    pair = tuple(eps) if isinstance(eps, (tuple, list)) else (eps, eps)
    if len(pair) != 2 or any(e is not None and not e >= 0 for e in pair):
        raise ValueError(f"eps must be None, a non-negative number, or two of these, got {eps}")
    return _ops().qk_norm_rope(q, k, positions, rope.axes_dims, rope.theta, rope.layout == "half", q_weight, k_weight,
                               [-1.0 if e is None else float(e) for e in pair])
