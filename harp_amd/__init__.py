"""harp_amd — MI355X (gfx950) ring-attention block for HARP's sequence-parallel attention.

Drop-in for HARP's ``libring_attention_ops.so`` (namespace ``ring_attention_ops``):
hand-written HIP kernels behind the C ABI of ``include/harp_ring_attn.h``
(``kernels/libharp_ra.so``) and a PyTorch-ROCm operator library
(``kernels/libring_attention_ops.so``).  The step before it, QK RMSNorm and the
rotary embedding, runs on the GPU too (``include/harp_qk_norm_rope.h``,
``kernels/libharp_async_op.so``, namespace ``async_op``), and
:class:`RingZAttention` wires projections, QK norm, RoPE, ring attention and
the output projection as the model's attention block does.  Around it
(``include/harp_block_ops.h``, ``kernels/libharp_block_ops.so``):
:func:`add_rms_norm`, the residual addition with its RMSNorm, and the Linear
layers in 8-bit integers for forward-only use (:class:`Int8Linear`,
:func:`quantize_attention`).  Build with ``python -m harp_amd.build``.
"""

from ._lib import (  # noqa: F401
    ABI_LIB,
    ASYNC_OPS_LIB,
    BLOCK_OPS_LIB,
    OPS_LIB,
    load_abi,
    load_async_ops,
    load_block_ops,
    load_ops,
)
from .ops import (  # noqa: F401
    RingAttention,
    abi_backward,
    abi_delta,
    abi_forward,
    backward_workspace_bytes,
    concat_chunks,
    forward_workspace_bytes,
    ring_attention,
)
from .qk import ApplyRotaryComplexFn, QKNormRopeFn, RMSNormFn  # noqa: F401
from .residual_norm import add_rms_norm, add_rms_norm_int8  # noqa: F401
from .int8 import Int8Linear, Int8Rows, int8_linear, quantize_attention, quantize_int8  # noqa: F401
from .attention import RingZAttention, project_qkv  # noqa: F401
from .wait_engine import CommWork, WaitEngine  # noqa: F401
from .gemm import xhblas_gemm  # noqa: F401

__version__ = "0.1.0"
