"""The attention block around the ring-attention operator, on the GPU.

:class:`RingZAttention` mirrors ``Z_Attention`` (src/models/z_image/module/
attn.py:51-105): it wraps the model's pretrained attention module (``to_q``,
``to_k``, ``to_v``, ``norm_q``, ``norm_k``, ``to_out``, ``heads``; the
``ZAttention`` of src/models/z_image/standalone_transformer.py:197-225) and
runs, for ``hidden_states`` [B, S, dim]:

1. the three projections, viewed as token-major [B, H, S, D] (attn.py:69-76);
2. QK RMSNorm and RoPE (attn.py:78-89), writing the token-major layout the
   ring kernel reads.  Steps 1-2 are one launch of the fused projection
   kernel (:mod:`harp_amd.qkv`) where it applies (head dim 128, no bias);
   otherwise plain library GEMMs (``nn.Linear``, hipBLASLt) and one fused
   norm + RoPE pass per tensor (:class:`QKNormRopeFn`), or the separate
   operator when only one of the two applies;
3. :class:`RingAttention` over ``sp_size`` KV chunks of the sequence (all on
   this GPU), then ``transpose(1, 2).flatten(2, 3)`` and ``to_out``
   (attn.py:99-103).

A module whose projections are :class:`harp_amd.Int8Linear`
(:func:`harp_amd.quantize_attention`) runs them in 8-bit integers, forward
only; ``hidden_states`` may then be 8-bit rows (:class:`harp_amd.Int8Rows`),
as :func:`harp_amd.add_rms_norm_int8` writes them.

The rotation may be given as positions along several axes
(:class:`harp_amd.AxialPositions`) instead of a complex table, and a module with
low-rank adapters beside its projections (:func:`harp_amd.adapt_attention`) takes
``requests``, which say whose tokens take which adapter.

``attn_mask`` is accepted and ignored, as in the reference (attn.py:91-97).
:func:`project_qkv` is steps 1-2 on their own (the producer of q, k, v).
"""

from __future__ import annotations

from types import SimpleNamespace
from typing import Optional, Tuple, Union

import torch
from torch import nn

from .adapters import (AdapterRequests, add_adapters, fused_adapters_arguments, is_adapted,
                       project_qkv_adapters, short_requests)
from .int8 import Int8Linear, Int8Rows, fused_int8_supported, is_int8, project_qkv_int8, quantize_int8
from .ops import RingAttention
from .qk import ApplyRotaryComplexFn, QKNormRopeFn, RMSNormFn
from .qkv import HEAD_DIM, ProjectQKVFn, fused_supported, qkv_project
from .rope import AxialPositions, AxialRope, qk_norm_axial_rope


def _norm_rope(x: torch.Tensor, norm: Optional[nn.Module], freqs_cis: Optional[torch.Tensor]) -> torch.Tensor:
    """RMSNorm (when ``norm`` is set) then RoPE (when ``freqs_cis`` is set) of a
    [B, H, S, D] view, on the async_op kernels (which take a token at least)."""
    if x.numel() == 0:
        return x
    if norm is not None:
        weight = getattr(norm, "weight", None)
        eps = float(norm.eps)
        if freqs_cis is not None:
            return QKNormRopeFn.apply(x, weight, freqs_cis, eps)
        return RMSNormFn.apply(x, weight, eps)
    if freqs_cis is not None:
        return ApplyRotaryComplexFn.apply(x, freqs_cis)
    return x


Freqs = Union[None, torch.Tensor, AxialPositions]


def _norms(attn) -> Tuple[Optional[nn.Module], Optional[nn.Module]]:
    return getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)


def _norm_axial_rope(attn, query: torch.Tensor, key: torch.Tensor, freqs: AxialPositions):
    """The QK RMSNorms where the module has them, and the rotation, q and k in one launch."""
    nq, nk = _norms(attn)
    return qk_norm_axial_rope(query, key, freqs.positions, freqs.rope, getattr(nq, "weight", None),
                              getattr(nk, "weight", None),
                              tuple(None if n is None else float(n.eps) for n in (nq, nk)))


def _records_gradient(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _project_short(attn, x: torch.Tensor, freqs: Freqs, requests: AdapterRequests):
    """What the one launch with adapters computes, for many short requests and without a gradient: its parts, in
    float32 to the end and rounded once as there, so that a token's result does not depend on how many requests are
    served with it."""
    def project(module):
        weight = module.base.weight
        y = torch.mm(x.flatten(0, 1), weight.t(), out_dtype=torch.float32).view(*x.shape[:2], weight.size(0))
        return add_adapters(y, x, module.adapters, requests).unflatten(-1, (attn.heads, -1)).transpose(1, 2)

    query, key, value = project(attn.to_q), project(attn.to_k), project(attn.to_v)
    if isinstance(freqs, AxialPositions):
        query, key = _norm_axial_rope(attn, query, key, freqs)
    else:  # the norms alone: no token is turned
        still = torch.zeros((x.size(1), 1), device=x.device)

        def normed(t, norm):
            if norm is None:
                return t
            return qk_norm_axial_rope(t, None, still, AxialRope((HEAD_DIM,), 1.0), norm.weight, eps=float(norm.eps))[0]

        query, key = (normed(t, n) for t, n in zip((query, key), _norms(attn)))
    if isinstance(freqs, torch.Tensor):
        turn = freqs.unsqueeze(-3)  # of all heads

        def rotate(t):
            return torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (-1, 2))) * turn).flatten(-2)

        query, key = rotate(query), rotate(key)
    # (token-major, as the one launch gives them)
    return tuple(t.transpose(1, 2).to(torch.bfloat16, memory_format=torch.contiguous_format).transpose(1, 2)
                 for t in (query, key, value))


def _project_bare(attn, hidden_states: Union[torch.Tensor, Int8Rows], freqs: Freqs):
    """The one launch for a module with adapters that no request takes (no ``requests``), or None where there is none.
    With a table, or no rotation, the call of the module without adapters; with positions the call of requests without
    an adapter, whose results those are (rounded, where the plain producer truncates behind norm and rotation)."""
    if isinstance(freqs, AxialPositions):
        if not isinstance(hidden_states, torch.Tensor):
            return None
        nobody = AdapterRequests(torch.full((1,), -1, dtype=torch.int32, device=hidden_states.device))
        arguments = fused_adapters_arguments(attn, hidden_states, freqs, nobody)
        if arguments is None:
            return None
        x, weights, a, b, *more = arguments  # (the adapters take no part, in a gradient either)
        return project_qkv_adapters((x, weights, [t.detach() for t in a], [t.detach() for t in b], *more))
    to = [m.base if is_adapted(m) else m for m in (attn.to_q, attn.to_k, attn.to_v)]
    nq, nk = _norms(attn)
    bare = SimpleNamespace(heads=attn.heads, norm_q=nq, norm_k=nk, to_q=to[0], to_k=to[1], to_v=to[2])
    if is_int8(bare):
        return project_qkv(bare, hidden_states, freqs) if fused_int8_supported(bare, freqs) else None
    if isinstance(hidden_states, torch.Tensor) and fused_supported(bare, hidden_states, freqs):
        return project_qkv(bare, hidden_states, freqs)
    return None


def _project_adapted(attn, hidden_states: Union[torch.Tensor, Int8Rows], freqs: Freqs,
                     fused: bool, requests: Optional[AdapterRequests]
                     ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """project_qkv of a module with adapters."""
    if fused and requests is None:
        bare = _project_bare(attn, hidden_states, freqs)
        if bare is not None:
            return bare
    if fused and requests is not None:
        arguments = fused_adapters_arguments(attn, hidden_states, freqs, requests)
        if arguments is not None:
            x, weights, a, b, _, _, _, norm_weights = arguments[:8]
            table = freqs if isinstance(freqs, torch.Tensor) else None
            if short_requests(x, requests) and not _records_gradient(x, *weights, *a, *b, *norm_weights, table):
                return _project_short(attn, x, freqs, requests)
            return project_qkv_adapters(arguments)
    x, heads, rows = hidden_states, attn.heads, None
    bases = [m.base if is_adapted(m) else m for m in (attn.to_q, attn.to_k, attn.to_v)]
    int8 = [isinstance(m, Int8Linear) for m in bases]
    if isinstance(x, Int8Rows):
        if not all(int8):
            raise ValueError("8-bit hidden states need 8-bit projections (harp_amd.quantize_attention)")
        rows, x = x, x.dequantize() if requests is not None else x
    elif any(int8):
        rows = quantize_int8(x)  # once for all three

    def project(module, quantised):
        y = module(rows if quantised else x)
        if requests is not None and is_adapted(module):
            y = add_adapters(y, x, module.adapters, requests)
        return y.unflatten(-1, (heads, -1)).transpose(1, 2)

    query, key, value = (project(m, i) for m, i in zip((attn.to_q, attn.to_k, attn.to_v), int8))
    if isinstance(freqs, AxialPositions):
        query, key = _norm_axial_rope(attn, query, key, freqs)
    else:
        nq, nk = _norms(attn)
        query, key = _norm_rope(query, nq, freqs), _norm_rope(key, nk, freqs)
    return query, key, value


def project_qkv(attn: nn.Module, hidden_states: Union[torch.Tensor, Int8Rows], freqs_cis: Freqs, fused: bool = True,
                requests: Optional[AdapterRequests] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k, v as token-major [B, H, S, D] views: projections, then QK RMSNorm
    and RoPE (attn.py:69-89).  With ``fused`` (default) and a module and input
    the fused kernel takes (:func:`harp_amd.qkv.fused_supported`: head dim
    128, no bias), all of it is one launch (:class:`ProjectQKVFn`); otherwise
    three library GEMMs and the separate norm + RoPE kernels.  With 8-bit
    projections the one launch is :func:`harp_amd.int8.project_qkv_int8` where
    it applies, else three 8-bit products and the separate kernels.

    ``freqs_cis`` may be positions along several axes
    (:class:`harp_amd.AxialPositions`): the one-launch forms read their table,
    otherwise :func:`harp_amd.qk_norm_axial_rope` norms and rotates q and k.
    ``requests``: which tokens take which of the module's adapters
    (:func:`harp_amd.adapt_attention`); without it none is added.  q and k of an
    adapted module are rounded to nearest where ``requests`` or positions are
    given; with a table and no requests they are the plain module's, which follow the
    reference and truncate."""
    adapted = any(is_adapted(getattr(attn, n, None)) for n in ("to_q", "to_k", "to_v"))
    if requests is not None and not adapted and not _adapted_out(attn):
        raise ValueError("requests need an attention module with adapters (harp_amd.adapt_attention)")
    if adapted:
        return _project_adapted(attn, hidden_states, freqs_cis, fused, requests)
    axial = freqs_cis if isinstance(freqs_cis, AxialPositions) else None
    if axial is not None:
        # the one-launch forms: neighbouring pairs of heads of 128 features
        fused = fused and axial.rope.layout == "interleaved" and axial.rope.dim == HEAD_DIM
        freqs_cis = axial.table() if fused else None
    if is_int8(attn):
        if not isinstance(hidden_states, Int8Rows):
            hidden_states = quantize_int8(hidden_states)  # once for all three
        if fused and fused_int8_supported(attn, freqs_cis):
            return project_qkv_int8(attn, hidden_states, freqs_cis)
    elif isinstance(hidden_states, Int8Rows):
        raise ValueError("8-bit hidden states need 8-bit projections (harp_amd.quantize_attention)")
    elif fused and fused_supported(attn, hidden_states, freqs_cis):
        nq, nk = getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)
        args = (hidden_states, attn.to_q.weight, attn.to_k.weight, attn.to_v.weight,
                None if nq is None else nq.weight, None if nk is None else nk.weight, freqs_cis,
                0.0 if nq is None else float(nq.eps), 0.0 if nk is None else float(nk.eps))
        if torch.is_grad_enabled() and any(isinstance(a, torch.Tensor) and a.requires_grad for a in args):
            return ProjectQKVFn.apply(*args)
        # no gradient can be taken: the kernel alone, without the pre-norm
        # products and rms a backward would need
        (q, k, v), _, _ = qkv_project(args[0], args[1:4], [(args[4], args[7]), (args[5], args[8]), (None, 0.0)],
                                      freqs_cis)
        return q, k, v
    heads = attn.heads
    query = attn.to_q(hidden_states).unflatten(-1, (heads, -1)).transpose(1, 2)
    key = attn.to_k(hidden_states).unflatten(-1, (heads, -1)).transpose(1, 2)
    value = attn.to_v(hidden_states).unflatten(-1, (heads, -1)).transpose(1, 2)
    if axial is not None:
        query, key = _norm_axial_rope(attn, query, key, axial)
        return query, key, value
    query = _norm_rope(query, getattr(attn, "norm_q", None), freqs_cis)
    key = _norm_rope(key, getattr(attn, "norm_k", None), freqs_cis)
    return query, key, value


def _adapted_out(attn) -> bool:
    to_out = getattr(attn, "to_out", None)
    return to_out is not None and len(to_out) > 0 and is_adapted(to_out[0])


class RingZAttention(nn.Module):
    """GPU drop-in for ``Z_Attention(pretrained_attn, sp_size)`` (attn.py:51-105).

    All ``sp_size`` ring chunks of the sequence are on this GPU: the sequence
    length S must be a multiple of ``sp_size``, and chunk c holds tokens
    c*S/sp_size .. (c+1)*S/sp_size - 1.  The result equals the reference's
    per-rank outputs concatenated over the ranks.
    """

    def __init__(self, pretrained_attn: nn.Module, sp_size: int):
        super().__init__()
        self.attn = pretrained_attn
        self.sp_size = sp_size

    def forward(self, hidden_states: Union[torch.Tensor, Int8Rows], RoPE_embeds: Freqs,
                attn_mask: Optional[torch.Tensor] = None, requests: Optional[AdapterRequests] = None) -> torch.Tensor:
        attn = self.attn
        tokens = (hidden_states.values if isinstance(hidden_states, Int8Rows) else hidden_states).size(1)
        if tokens % self.sp_size:
            raise ValueError(f"sequence length {tokens} is not a multiple of sp_size {self.sp_size}")
        query, key, value = project_qkv(attn, hidden_states, RoPE_embeds, requests=requests)
        out = RingAttention.apply(query, key, value, self.sp_size).transpose(1, 2).flatten(2, 3)
        out = attn.to_out[0](out, requests) if _adapted_out(attn) else attn.to_out[0](out)
        if len(attn.to_out) > 1:  # dropout / identity
            out = attn.to_out[1](out)
        return out
