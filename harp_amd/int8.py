"""Linear layers in 8-bit integers, on the GPU, for forward-only use.

Activations and weights are :class:`Int8Rows`: int8 values with one float32
scale for each row (each token of the activations, each output feature of a
weight)::

    scale = max |row| / 127,   values = row / scale to nearest, ties to even

A row of zeros has scale 0; a row that holds an infinity or a NaN has scale
NaN, so that every result it reaches is NaN.  :func:`int8_linear` multiplies
two sets of rows on the matrix cores, exactly in 32-bit integers, and applies
the scales and the bias in its epilogue.

:class:`Int8Linear` stands in for an ``nn.Linear``: it keeps the weight's rows
and quantises its input, unless that comes as rows already
(:func:`harp_amd.add_rms_norm_int8` writes them).  :func:`quantize_attention`
replaces the projections of the model's attention module, which
:func:`harp_amd.project_qkv` and :class:`harp_amd.RingZAttention` then run on:
q, k and v in one launch, with the QK RMSNorm and RoPE in its epilogue where
the heads have 128 features.

No gradient is recorded: where one would be, or an argument carries a
forward-mode tangent, the functions raise.  There is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import nn

from . import _lib

HEAD_DIM = 128


_harp_block = None


def _ops():
    """torch.ops.harp_block, its library loaded at the first call."""
    global _harp_block
    if _harp_block is None:
        _lib.load_block_ops()
        _harp_block = torch.ops.harp_block
    return _harp_block


def _refuse_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is forward only: call it under torch.no_grad(), or on tensors that need no gradient")


class Int8Rows(NamedTuple):
    """8-bit rows: ``values`` int8 [.., C], ``scales`` float32 [..].

    Row r stands for ``values[r] * scales[r]``.  The kernels take rows that
    start at multiples of 16 bytes, as the functions here lay them out (views
    of whole rows, or of their first columns, keep that)."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """values * scales as a bfloat16 or float32 tensor."""
        _refuse_grad("Int8Rows.dequantize", self.scales)
        return _ops().dequantize_int8(self.values, self.scales, dtype)


def quantize_int8(x: torch.Tensor) -> Int8Rows:
    """8-bit rows of a bfloat16 or float32 tensor [.., C], C up to 32768."""
    _refuse_grad("quantize_int8", x)
    return Int8Rows(*_ops().quantize_int8(x))


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x [.., K] times the transpose of weight [N, K], plus bias [N]: a
    bfloat16 or float32 tensor [.., N].  K up to 65536."""
    _refuse_grad("int8_linear", x.scales, weight.scales, bias)
    if weight.values.size(-1) != x.values.size(-1):
        raise RuntimeError(f"weight must be [N, {x.values.size(-1)}], got {tuple(weight.values.shape)}")
    return _ops().linear_int8(x.values, x.scales, weight.values, weight.scales, bias, out_dtype)


def _weight_row_bytes(cols: int) -> int:
    """Bytes of a row of a module's weight: whole 128-byte cache lines for long rows, so that a
    tile's 128 bytes of a row are one line (1333 tokens x 1001 features of 2570 columns: 12.6 us
    instead of 14.6)."""
    unit = 16 if cols < 1024 else 128
    return -(-cols // unit) * unit


class Int8Linear(nn.Module):
    """An ``nn.Linear`` with its weight in 8-bit rows, forward only.

    ``weight_values`` holds the rows padded to multiples of 16 bytes (128 from
    1024 columns on), ``weight_scales`` their scales (float32, also where the
    module's other tensors are converted to 16 bits: convert before quantising)."""

    def __init__(self, weight: Int8Rows, bias: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        values, scales = weight
        if values.dim() != 2 or values.dtype != torch.int8 or scales.shape != values.shape[:1]:
            raise ValueError(f"weight must be int8 rows [N, K] with N scales, got {values.dtype} {tuple(values.shape)} "
                             f"and {tuple(scales.shape)}")
        if scales.dtype != torch.float32:
            raise ValueError(f"weight scales must be float32, got {scales.dtype}")
        if bias is not None and bias.shape != values.shape[:1]:
            raise ValueError(f"bias must be [{values.size(0)}], got {tuple(bias.shape)}")
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
        self.out_features, self.in_features = values.shape
        self.out_dtype = out_dtype
        store = torch.zeros((values.size(0), _weight_row_bytes(values.size(1))), dtype=torch.int8, device=values.device)
        store[:, :self.in_features] = values
        self.register_buffer("weight_values", store)
        self.register_buffer("weight_scales", scales.detach().clone())
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_quantized(cls, values: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       out_dtype: torch.dtype = torch.bfloat16) -> "Int8Linear":
        """From int8 values [N, K] in any layout and float32 scales [N]."""
        return cls(Int8Rows(values, scales), bias, out_dtype)

    @classmethod
    def from_linear(cls, linear: nn.Linear, out_dtype: torch.dtype = torch.bfloat16) -> "Int8Linear":
        """From an ``nn.Linear`` (or a module with its ``weight`` and ``bias``) on a HIP device."""
        return cls(quantize_int8(linear.weight.detach()), getattr(linear, "bias", None), out_dtype)

    @property
    def weight(self) -> Int8Rows:
        """The weight's 8-bit rows [N, K]."""
        return Int8Rows(self.weight_values[:, :self.in_features], self.weight_scales)

    def forward(self, x: Union[torch.Tensor, Int8Rows]) -> torch.Tensor:
        rows = isinstance(x, Int8Rows)
        features = (x.values if rows else x).size(-1)
        if features != self.in_features:
            raise RuntimeError(f"Int8Linear of {self.in_features} features got rows of {features}")
        # the operators read the weight's first in_features columns
        if rows:
            _refuse_grad("Int8Linear", x.scales)
            return _ops().linear_int8(x.values, x.scales, self.weight_values, self.weight_scales, self.bias,
                                      self.out_dtype, self.in_features)
        _refuse_grad("Int8Linear", x)
        return _ops().linear_int8_dynamic(x, self.weight_values, self.weight_scales, self.bias, self.out_dtype,
                                          self.in_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class Int8Attention(nn.Module):
    """The attributes :func:`harp_amd.project_qkv` and
    :class:`harp_amd.RingZAttention` read of the model's attention module,
    with the projections in 8 bits."""

    def __init__(self, attn: nn.Module):
        super().__init__()
        self.heads = attn.heads
        self.to_q, self.to_k, self.to_v = (Int8Linear.from_linear(m) for m in (attn.to_q, attn.to_k, attn.to_v))
        self.norm_q, self.norm_k = getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)
        to_out = getattr(attn, "to_out", None)
        if to_out is not None:
            self.to_out = nn.ModuleList([Int8Linear.from_linear(to_out[0]), *to_out[1:]])


def quantize_attention(attn: nn.Module) -> Int8Attention:
    """The attention module with ``to_q``, ``to_k``, ``to_v`` and ``to_out[0]``
    as :class:`Int8Linear`; its norms are shared, its weights copied."""
    return Int8Attention(attn)


def is_int8(attn) -> bool:
    """True when the module's q, k and v projections are all :class:`Int8Linear`."""
    return all(isinstance(getattr(attn, n, None), Int8Linear) for n in ("to_q", "to_k", "to_v"))


def fused_int8_supported(attn, freqs_cis: Optional[torch.Tensor]) -> bool:
    """True when :func:`project_qkv_int8` takes the module: heads of 128
    features, no bias, bf16 outputs, and RoPE only with both norms' weights."""
    lins = (attn.to_q, attn.to_k, attn.to_v)
    if any(m.bias is not None or m.out_dtype != torch.bfloat16 or m.out_features != attn.heads * HEAD_DIM
           or m.in_features != lins[0].in_features for m in lins):
        return False
    norms = [getattr(attn, "norm_q", None), getattr(attn, "norm_k", None)]
    weights = [None if nm is None else getattr(nm, "weight", None) for nm in norms]
    if any(nm is not None and w is None for nm, w in zip(norms, weights)):
        return False
    return freqs_cis is None or all(w is not None for w in weights)


def project_qkv_int8(attn, rows: Int8Rows, freqs_cis: Optional[torch.Tensor]
                     ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k, v [B, H, S, 128] (token-major strides) of 8-bit rows [B, S, dim],
    in one launch: the products, the QK RMSNorm of q and k and their RoPE, in
    float32 with one rounding at the end."""
    norms = [getattr(attn, "norm_q", None), getattr(attn, "norm_k", None), None]
    weights = [None if nm is None else nm.weight for nm in norms]
    _refuse_grad("project_qkv with 8-bit projections", rows.scales, *weights)
    w = [m.weight for m in (attn.to_q, attn.to_k, attn.to_v)]
    q, k, v = _ops().qkv_int8(rows.values, rows.scales, [r.values for r in w], [r.scales for r in w], weights,
                              [0.0 if nm is None else float(nm.eps) for nm in norms], freqs_cis)
    return q, k, v
