"""Low-rank adapters of many requests at once beside shared projections, on the GPU.

An adapter of rank r adds ``scale * (x A^T) B^T`` to a projection's result, A [r, in] and
B [out, r].  A batch holds many requests with an adapter each, or none, of n that are kept
stacked (:class:`Adapters`); :class:`AdapterRequests` says which tokens are whose.
:func:`add_adapters` adds each token's own adapter in one or two launches, differentiable
(any number of the adapters may be trained at once, the projection's weight stays
frozen or trains by itself).  :class:`AdaptedLinear` puts adapters beside an
``nn.Linear`` or an :class:`harp_amd.Int8Linear`, :func:`adapt_attention` beside
the projections of the model's attention module, which :func:`harp_amd.project_qkv`
and :class:`harp_amd.RingZAttention` then run with ``requests``.

Which request takes which adapter is read on the GPU only: a call neither waits for
the device nor depends on the values, so a captured graph may be replayed with others.

An infinity or a NaN in one adapter reaches no token of the requests that do not take it.

Tokens and adapters are bfloat16; a projection's result is bfloat16, or float32 where no
gradient is taken.  Sums are float32, the result is rounded once.  There is no CPU path.
"""

from __future__ import annotations

from types import SimpleNamespace
from typing import NamedTuple, Optional, Union

import torch
import torch.nn.functional as F
from torch import nn

from .int8 import Int8Linear, Int8Rows
from .qkv import HEAD_DIM, fused_supported
from .rope import AxialPositions, _ops


MAX_TOKENS = 1 << 25  # of one call of the adapters' kernels


class Adapters(NamedTuple):
    """n adapters of one rank (1 to 128) beside one projection: ``a`` bfloat16 [n, rank, in],
    ``b`` bfloat16 [n, out, rank], ``scales`` float32 [n] or None for ones.  Adapters of
    different ranks are stacked with zeros behind the shorter ones."""

    a: torch.Tensor
    b: torch.Tensor
    scales: Optional[torch.Tensor] = None


class AdapterRequests(NamedTuple):
    """Which tokens take which adapter, on the device, int32 or int64.

    ``index`` [R]: the adapter of each request; one that is not 0 .. n - 1 takes none.
    ``offsets`` [R + 1], never falling: request i is tokens offsets[i] .. offsets[i + 1] - 1 of all
    tokens in a row ([B, S] flattened); the others take no adapter.  None: all requests have
    the same number of tokens, as the rows of a batch have."""

    index: torch.Tensor
    offsets: Optional[torch.Tensor] = None


def add_adapters(base: torch.Tensor, x: torch.Tensor, adapters: Adapters, requests: AdapterRequests) -> torch.Tensor:
    """base + scale * (x A^T) B^T of each token's adapter.

    base [.., out] is the projection of x [.., in]; the result is a new tensor of base's type.
    Gradients of base (bfloat16), x and the adapters' a and b, once and in reverse mode."""
    return _ops().add_adapters(base, x, adapters.a, adapters.b, adapters.scales, requests.index, requests.offsets)


class AdaptedLinear(nn.Module):
    """A Linear layer with adapters beside it.

    ``base``: an ``nn.Linear`` (or a module with its ``weight`` and ``bias``) or an
    :class:`harp_amd.Int8Linear`, shared by all requests.  The adapters' a and b become
    parameters over the same memory (kept as they are if they are parameters); the scales are
    a buffer that stays float32 where the module is cast to another type."""

    def __init__(self, base, adapters: Adapters):
        super().__init__()
        a, b, scales = adapters
        if a.dim() != 3 or b.dim() != 3 or b.size(0) != a.size(0) or b.size(2) != a.size(1):
            raise ValueError(f"adapters must be a [n, rank, in] and b [n, out, rank], got {tuple(a.shape)} and "
                             f"{tuple(b.shape)}")
        weight = base.weight.values if isinstance(base, Int8Linear) else base.weight
        if weight.shape != (b.size(1), a.size(2)):
            raise ValueError(f"adapters from {a.size(2)} to {b.size(1)} features beside a weight {tuple(weight.shape)}")
        if scales is not None and (scales.dtype != torch.float32 or scales.shape != a.shape[:1]):
            raise ValueError(f"scales must be float32 [{a.size(0)}], got {scales.dtype} {tuple(scales.shape)}")
        self.base = base

        def parameter(t):
            return t if isinstance(t, nn.Parameter) else nn.Parameter(t, requires_grad=t.requires_grad)

        self.a, self.b = parameter(a), parameter(b)
        self.register_buffer("scales", scales)

    def _apply(self, fn, *args, **kwargs):
        scales = self.scales
        super()._apply(fn, *args, **kwargs)
        # the scales stay float32 where the module is cast (``module.to(torch.bfloat16)``)
        if scales is not None and self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    @property
    def adapters(self) -> Adapters:
        return Adapters(self.a, self.b, self.scales)

    def forward(self, x: Union[torch.Tensor, Int8Rows], requests: Optional[AdapterRequests] = None) -> torch.Tensor:
        """The projection of x, plus each request's adapter; without ``requests`` the projection alone."""
        base = self.base
        if callable(base):
            y = base(x)
        else:
            y = F.linear(x, base.weight, getattr(base, "bias", None))
        if requests is None:
            return y
        return add_adapters(y, x.dequantize() if isinstance(x, Int8Rows) else x, self.adapters, requests)

    def extra_repr(self) -> str:
        return f"adapters={self.a.size(0)}, rank={self.a.size(1)}"


class AdaptedAttention(nn.Module):
    """The attributes :func:`harp_amd.project_qkv` and :class:`harp_amd.RingZAttention` read of the
    model's attention module, with adapters beside its projections."""

    def __init__(self, attn, **adapters: Optional[Adapters]):
        super().__init__()
        self.heads = attn.heads
        for name in ("to_q", "to_k", "to_v"):
            low = adapters.get(name)
            setattr(self, name, getattr(attn, name) if low is None else AdaptedLinear(getattr(attn, name), low))
        self.norm_q, self.norm_k = getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)
        to_out, low = getattr(attn, "to_out", None), adapters.get("to_out")
        if to_out is not None:
            self.to_out = nn.ModuleList([to_out[0] if low is None else AdaptedLinear(to_out[0], low), *to_out[1:]])
        elif low is not None:
            raise ValueError("to_out adapters need an attention module with to_out")


def adapt_attention(attn, to_q: Optional[Adapters] = None, to_k: Optional[Adapters] = None,
                    to_v: Optional[Adapters] = None, to_out: Optional[Adapters] = None) -> AdaptedAttention:
    """The attention module with adapters beside ``to_q``, ``to_k``, ``to_v`` and ``to_out[0]`` where
    given; its projections and norms are shared.  A module of :func:`harp_amd.quantize_attention`
    keeps its projections in 8 bits."""
    return AdaptedAttention(attn, to_q=to_q, to_k=to_k, to_v=to_v, to_out=to_out)


def _tokens(hidden_states: torch.Tensor) -> int:
    return hidden_states.numel() // max(hidden_states.size(-1), 1)


def fused_adapters_arguments(attn, hidden_states: torch.Tensor, freqs, requests: AdapterRequests) -> Optional[tuple]:
    """What :func:`project_qkv_adapters` takes for this module and input, or None where it does not: adapters of one
    number and one rank, a multiple of 8, beside bfloat16 projections without a bias, heads of 128 features, norms of
    both q and k with a rotation, positions along interleaved axes where a gradient is recorded, and 2^25 tokens at
    most."""
    lins = (attn.to_q, attn.to_k, attn.to_v)
    if not all(is_adapted(m) for m in lins) or not isinstance(hidden_states, torch.Tensor):
        return None
    bases = [m.base for m in lins]
    if any(isinstance(m, Int8Linear) for m in bases) or _tokens(hidden_states) > MAX_TOKENS:
        return None
    a, b = [m.a for m in lins], [m.b for m in lins]
    if a[1].shape != a[0].shape or a[2].shape != a[0].shape or a[0].size(1) % 8:
        return None
    if b[1].shape != b[0].shape or b[2].shape != b[0].shape:
        return None
    device = hidden_states.device
    for t in (*a, *b):
        if not t.is_contiguous() or t.dtype != torch.bfloat16 or t.device != device or t.data_ptr() % 16:
            return None
    norms = [getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)]
    norm_weights = [getattr(n, "weight", None) for n in norms]
    axial = isinstance(freqs, AxialPositions)
    if axial:
        rope = freqs.rope
        if rope.layout != "interleaved" or rope.dim != HEAD_DIM or norm_weights[0] is None or norm_weights[1] is None:
            return None
    elif freqs is not None and freqs.dtype != torch.complex64:
        return None
    bare = SimpleNamespace(heads=attn.heads, norm_q=norms[0], norm_k=norms[1], to_q=bases[0], to_k=bases[1],
                           to_v=bases[2])
    if not fused_supported(bare, hidden_states, None if axial else freqs):
        return None
    weights = [m.weight for m in bases]
    if not axial and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (hidden_states, *norm_weights, *a, *b, *weights)):
        return None
    eps = [0.0 if n is None else float(n.eps) for n in norms]
    rotation = (None, freqs.positions, rope.axes_dims, rope.theta) if axial else (freqs, None, (), ())
    return (hidden_states, weights, a, b, [m.scales for m in lins], requests.index, requests.offsets, norm_weights, eps,
            *rotation)


def project_qkv_adapters(arguments: tuple):
    """q, k, v [B, H, S, 128] (token-major strides) of a module with adapters beside all three projections: one
    launch for x A^T, one for the products, the adapters, the QK RMSNorm and the rotation."""
    q, k, v = _ops().qkv_adapters(*arguments)
    return q, k, v


def short_requests(hidden_states: torch.Tensor, requests: AdapterRequests) -> bool:
    """Whether the parts of the one launch, in float32, serve these requests sooner: more than 8 of them, with fewer
    than 8 tokens on the average.  The contraction takes a tile more for each request among a block's tokens, 128 or
    256 of them.  30 heads from 3840 features, one launch and parts: rank 16, 9 requests of one token 64 and 63 us, 32
    of one token 116 and 78, 64 of four 128 and 124; rank 128, 9 of one token 136 and 85, 64 of four 403 and 242."""
    count = requests.index.numel()
    return count > 8 and _tokens(hidden_states) < 8 * count


def is_adapted(module) -> bool:
    return isinstance(module, AdaptedLinear)
