"""The q/k/v producer's block of 160 tokens x 2 heads (launch_proj in
harp_amd/csrc/proj_kernels.hip): ten waves, of which eight copy one row group of a
weight tile less than the others.  It sums in the same order as the other blocks,
so its outputs equal, bit for bit, those of the same tokens in a call long enough
for 256-token blocks, and the fp64 product to the bound of tests/test_gpu_qkv.py."""

import math

import pytest
import torch

from harp_amd import qkv
from tests.test_gpu_qkv import _check_product, _inputs

pytestmark = pytest.mark.gpu

CUS = 256


def _block(S, heads, n_outs):
    """tokens of a block: the smallest of these of which one round holds the whole call"""
    return next((t for t in (128, 160, 256) if n_outs * math.ceil(S / t) * ((heads + 1) // 2) <= CUS), 0)


@pytest.mark.parametrize("S,dim,heads,n_outs", [
    (768, 64, 30, 3),     # one k-tile
    (641, 192, 29, 3),    # three, one token in the last block and half a last pair
    (1100, 128, 23, 3),
    (1900, 320, 42, 1),   # one output
    (641, 448, 49, 2),    # seven k-tiles: past the three stages
])
def test_blocks_of_160_tokens_equal_large_blocks(S, dim, heads, n_outs):
    assert torch.cuda.get_device_properties(0).multi_processor_count == CUS
    assert _block(S, heads, n_outs) == 160
    x, ws, norms, fc, _ = _inputs(1, S, dim, heads, "bf16", True, False, seed=S + dim)
    norms = (norms + [(None, 0.0)])[:n_outs]
    got = qkv.qkv_project(x, ws[:n_outs], norms, fc, keep_for_backward=True)
    B = next(b for b in range(2, 64) if _block(b * S, heads, n_outs) in (0, 256))
    want = qkv.qkv_project(x.expand(B, S, dim).contiguous(), ws[:n_outs], norms, fc, keep_for_backward=True)
    torch.cuda.synchronize()
    for i in range(n_outs):
        for b in (0, B - 1):
            assert torch.equal(got[0][i][0], want[0][i][b])
            if norms[i][0] is not None:
                assert torch.equal(got[1][i][0], want[1][i][b])
                assert torch.equal(got[2][i].view(heads, S), want[2][i].view(B, heads, S)[b])
        _check_product(x, ws[i], got[0][i] if norms[i][0] is None else got[1][i], f"out {i}")
