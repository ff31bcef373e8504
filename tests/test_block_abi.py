"""CPU tests of the boundary of the operators around the attention block:
libharp_ra.so exports exactly the functions include/harp_block_ops.h declares,
bad arguments are refused on the host before any device call, and the Python
entry points refuse what they do not take (no GPU needed)."""

import os
import re
import subprocess

import pytest
import torch
from torch import nn

import harp_amd
from harp_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "harp_block_ops.h")
FAKE = 1 << 20  # aligned, never dereferenced: validation fails first
EINVAL, EUNSUPPORTED, ENOMEM = 1, 2, 3
F32, BF16 = _lib.HARP_BLK_F32, _lib.HARP_BLK_BF16


def header_functions():
    text = open(HEADER).read()
    return sorted(set(re.findall(r"HARP_BLK_API\s+[\w\s\*]+?\b(harp_blk_\w+)\s*\(", text)))


def test_header_prototypes_and_exports_agree():
    fns = header_functions()
    assert len(fns) == 9 and set(fns) == set(_lib.BLK_PROTOTYPES)
    nm = subprocess.run(["nm", "-D", "--defined-only", str(_lib.ABI_LIB)], capture_output=True, text=True)
    exported = {ln.split()[-1] for ln in nm.stdout.splitlines() if " T " in ln}
    assert {s for s in exported if s.startswith("harp_blk_")} == set(fns)


def _err():
    return harp_amd.load_abi().harp_blk_last_error().decode()


FWD = dict(x=FAKE, ldx=64, xd=BF16, r=FAKE, ldr=64, rd=BF16, w=FAKE, wd=BF16, eps=1e-5, y=FAKE, ldy=64, h=FAKE, ldh=64,
           rstd=FAKE, rows=4, cols=64)


def _fwd(fn, over):
    a = {**FWD, **over}
    return fn(a["x"], a["ldx"], a["xd"], a["r"], a["ldr"], a["rd"], a["w"], a["wd"], a["eps"], a["y"], a["ldy"], a["h"],
              a["ldh"], a["rstd"], a["rows"], a["cols"], None)


@pytest.mark.parametrize("over,code,msg", [
    (dict(x=None), EINVAL, "x is NULL"),
    (dict(x=FAKE + 1), EINVAL, "aligned"),
    (dict(xd=F32, x=FAKE + 2), EINVAL, "aligned"),
    (dict(xd=7), EINVAL, "dtype"),
    (dict(rd=7), EINVAL, "dtype"),
    (dict(wd=7), EINVAL, "dtype"),
    (dict(ldx=-1), EINVAL, "row stride"),
    (dict(ldy=63), EINVAL, "may not overlap"),
    (dict(ldh=0), EINVAL, "may not overlap"),
    (dict(r=None), EINVAL, "without a residual"),
    (dict(y=None), EINVAL, "y is NULL"),
    (dict(rows=-1), EINVAL, "rows"),
    (dict(cols=0), EINVAL, "cols"),
    (dict(cols=32769, ldx=32769), EUNSUPPORTED, "32768"),
    (dict(eps=-1.0), EINVAL, "eps"),
    (dict(eps=float("nan")), EINVAL, "eps"),
    (dict(rstd=FAKE + 2), EINVAL, "rstd"),
])
def test_norm_forward_refuses(over, code, msg):
    rc = _fwd(harp_amd.load_abi().harp_blk_add_rms_norm_forward, over)
    assert rc == code and msg in _err(), (rc, _err())


@pytest.mark.parametrize("over,code,msg", [
    (dict(y=FAKE + 8), EINVAL, "16-byte aligned"),       # q
    (dict(ldy=72), EINVAL, "multiple of 16"),            # ld_q
    (dict(cols=65, ldx=65, ldr=65, ldh=65, ldy=64), EINVAL, "multiple of 16 in [80"),
    (dict(rstd=None), EINVAL, "scales is NULL"),
])
def test_norm_int8_refuses(over, code, msg):
    a = {**FWD, **over}
    rc = harp_amd.load_abi().harp_blk_add_rms_norm_int8(
        a["x"], a["ldx"], a["xd"], a["r"], a["ldr"], a["rd"], a["w"], a["wd"], a["eps"], a["h"], a["ldh"], a["y"],
        a["ldy"], a["rstd"], a["rows"], a["cols"], None)
    assert rc == code and msg in _err(), (rc, _err())


def _bwd(**over):
    a = dict(dy=FAKE, ldy=64, xd=BF16, dh=FAKE, lddh=64, h=FAKE, ldh=64, hd=BF16, w=FAKE, wd=BF16, rstd=FAKE, dx=FAKE,
             lddx=64, dr=None, lddr=0, gw=FAKE, gwd=F32, rows=4, cols=64, ws=FAKE, wsb=1 << 20)
    a.update(over)
    return harp_amd.load_abi().harp_blk_add_rms_norm_backward(
        a["dy"], a["ldy"], a["xd"], a["dh"], a["lddh"], a["h"], a["ldh"], a["hd"], a["w"], a["wd"], a["rstd"], a["dx"],
        a["lddx"], a["dr"], a["lddr"], a["gw"], a["gwd"], a["rows"], a["cols"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,code,msg", [
    (dict(dy=None), EINVAL, "dy is NULL"),
    (dict(h=None), EINVAL, "h is NULL"),
    (dict(rstd=None), EINVAL, "rstd is NULL"),
    (dict(dx=None), EINVAL, "dx is NULL"),
    (dict(lddx=60), EINVAL, "may not overlap"),
    (dict(dr=FAKE, lddr=60), EINVAL, "may not overlap"),
    (dict(gwd=9), EINVAL, "dtype"),
    (dict(ws=None), ENOMEM, "workspace"),
    (dict(wsb=8), ENOMEM, "workspace"),
    (dict(ws=FAKE + 4), EINVAL, "workspace"),
])
def test_norm_backward_refuses(over, code, msg):
    rc = _bwd(**over)
    assert rc == code and msg in _err(), (rc, _err())


def test_workspace_sizes():
    lib = harp_amd.load_abi()
    assert lib.harp_blk_backward_workspace_bytes(1, 64) == 64 * 4
    big = lib.harp_blk_backward_workspace_bytes(1 << 20, 3840)
    assert big % (3840 * 4) == 0 and big <= 1024 * 3840 * 4
    assert lib.harp_blk_backward_workspace_bytes(4, 40000) == 2 ** 64 - 1


LIN = dict(x=FAKE, ldx=64, xs=FAKE, w=FAKE, ldw=64, ws=FAKE, b=None, bd=BF16, y=FAKE, ldy=32, yd=BF16, M=4, N=32, K=64)


@pytest.mark.parametrize("over,code,msg", [
    (dict(x=None), EINVAL, "x must"),
    (dict(x=FAKE + 8), EINVAL, "x must"),
    (dict(ldx=72), EINVAL, "multiple of 16"),
    (dict(ldx=48), EINVAL, "multiple of 16 in [64"),
    (dict(ldw=(1 << 22) + 16), EINVAL, "row stride"),
    (dict(xs=None), EINVAL, "x_scales"),
    (dict(ws=None), EINVAL, "w_scales"),
    (dict(b=FAKE, bd=5), EINVAL, "dtype"),
    (dict(y=FAKE + 1), EINVAL, "aligned"),
    (dict(ldy=31), EINVAL, "may not overlap"),
    (dict(yd=3), EINVAL, "dtype"),
    (dict(N=0), EINVAL, "positive"),
    (dict(K=0), EINVAL, "positive"),
    (dict(M=-1), EINVAL, "M=-1"),
    (dict(K=65537, ldx=65552, ldw=65552), EUNSUPPORTED, "65536"),
])
def test_linear_refuses(over, code, msg):
    a = {**LIN, **over}
    rc = harp_amd.load_abi().harp_blk_linear_int8(a["x"], a["ldx"], a["xs"], a["w"], a["ldw"], a["ws"], a["b"], a["bd"],
                                                  a["y"], a["ldy"], a["yd"], a["M"], a["N"], a["K"], None)
    assert rc == code and msg in _err(), (rc, _err())


@pytest.mark.parametrize("over,outs_over,code,msg", [
    (dict(N=200), {}, EUNSUPPORTED, "n_out"),
    (dict(K=0), {}, EINVAL, "k_dim"),
    (dict(x=FAKE + 1), {}, EINVAL, "x must"),
    (dict(n=0), {}, EINVAL, "outs"),
    (dict(n=4), {}, EINVAL, "outs"),
    (dict(f=FAKE + 4), {}, EINVAL, "freqs"),
    (dict(fss=130), {}, EINVAL, "freqs strides"),
    ({}, {1: dict(weight=None)}, EINVAL, "outs[1].weight"),
    ({}, {0: dict(ld_weight=100)}, EINVAL, "outs[0].weight"),
    ({}, {2: dict(weight_scales=None)}, EINVAL, "outs[2].weight_scales"),
    ({}, {2: dict(ld_y=128)}, EINVAL, "outs[2].y"),
    ({}, {0: dict(norm_weight_dtype=7)}, EINVAL, "dtype"),
    ({}, {0: dict(eps=-1.0)}, EINVAL, "eps"),
])
def test_qkv_refuses(over, outs_over, code, msg):
    outs = (_lib.BlkQkvOut * 3)()
    for o in outs:
        o.weight, o.ld_weight, o.weight_scales, o.y, o.ld_y = FAKE, 128, FAKE, FAKE, 256
        o.norm_weight, o.norm_weight_dtype, o.eps = FAKE, BF16, 1e-6
    for i, kv in outs_over.items():
        for k, v in kv.items():
            setattr(outs[i], k, v)
    a = dict(x=FAKE, ldx=128, xs=FAKE, B=1, S=8, K=128, N=256, f=FAKE, fsb=0, fss=128, n=3)
    a.update(over)
    rc = harp_amd.load_abi().harp_blk_qkv_int8(a["x"], a["ldx"], a["xs"], a["B"], a["S"], a["K"], a["N"], a["f"],
                                               a["fsb"], a["fss"], outs, a["n"], None)
    assert rc == code and msg in _err(), (rc, _err())


def test_empty_calls_do_nothing():
    lib = harp_amd.load_abi()
    assert _fwd(lib.harp_blk_add_rms_norm_forward, dict(rows=0)) == 0
    assert _bwd(rows=0) == 0
    a = {**LIN, "M": 0}
    assert lib.harp_blk_linear_int8(a["x"], a["ldx"], a["xs"], a["w"], a["ldw"], a["ws"], a["b"], a["bd"], a["y"],
                                    a["ldy"], a["yd"], a["M"], a["N"], a["K"], None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    rows = harp_amd.Int8Rows(torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3))
    for call in (lambda: harp_amd.add_rms_norm(x, x), lambda: harp_amd.add_rms_norm(x.requires_grad_(), None),
                 lambda: harp_amd.add_rms_norm_int8(x.detach(), None), lambda: harp_amd.quantize_int8(x.detach()),
                 lambda: rows.dequantize(), lambda: harp_amd.int8_linear(rows, rows),
                 lambda: harp_amd.Int8Linear(rows)(rows)):
        with pytest.raises(RuntimeError, match="HIP device only"):
            call()


def test_gradients_are_refused():
    x = torch.zeros(3, 64, dtype=torch.bfloat16, requires_grad=True)
    rows = harp_amd.Int8Rows(torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3))
    for call in (lambda: harp_amd.add_rms_norm_int8(x), lambda: harp_amd.quantize_int8(x),
                 lambda: harp_amd.Int8Linear(rows)(x),
                 lambda: harp_amd.int8_linear(rows, rows, torch.zeros(3, requires_grad=True))):
        with pytest.raises(RuntimeError, match="forward only"):
            call()


def test_int8_linear_module():
    """Layout, checks and state of the module (no kernel runs)."""
    values = torch.arange(-60, 60, dtype=torch.int8).view(5, 24)
    scales = torch.rand(5)
    lin = harp_amd.Int8Linear.from_quantized(values.t().contiguous().t(), scales, torch.ones(5))
    assert lin.weight_values.shape == (5, 32) and bool((lin.weight_values[:, 24:] == 0).all())
    assert torch.equal(lin.weight.values, values) and torch.equal(lin.weight.scales, scales)
    assert lin.weight.values.stride() == (32, 1)
    other = harp_amd.Int8Linear.from_quantized(torch.zeros_like(values), torch.zeros(5), torch.zeros(5))
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other.weight.values, values) and torch.equal(other.bias, torch.ones(5))
    for bad in (dict(values=values.float()), dict(scales=scales[:4]), dict(scales=scales.double()),
                dict(bias=torch.ones(4)), dict(out_dtype=torch.float16)):
        kw = {**dict(values=values, scales=scales, bias=None, out_dtype=torch.bfloat16), **bad}
        with pytest.raises(ValueError):
            harp_amd.Int8Linear.from_quantized(**kw)


def test_rows_need_8_bit_projections():
    attn = nn.Module()
    attn.heads = 1
    attn.to_q = attn.to_k = attn.to_v = nn.Linear(64, 128, bias=False).to(torch.bfloat16)
    rows = harp_amd.Int8Rows(torch.zeros(1, 3, 64, dtype=torch.int8), torch.zeros(1, 3))
    with pytest.raises(ValueError, match="8-bit projections"):
        harp_amd.project_qkv(attn, rows, None)


def test_gradients_of_scales_are_refused():
    values, scales = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3, requires_grad=True)
    rows, plain = harp_amd.Int8Rows(values, scales), harp_amd.Int8Rows(values, scales.detach())
    for call in (lambda: rows.dequantize(), lambda: harp_amd.int8_linear(rows, plain),
                 lambda: harp_amd.int8_linear(plain, rows), lambda: harp_amd.Int8Linear(plain)(rows)):
        with pytest.raises(RuntimeError, match="forward only"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device only"):
            call()


def _dual_calls(dual, plain):
    """Every operator with one argument made dual; plain gives an int8 [3, 64] and floats."""
    f, q, s, w, ops = plain["f"], plain["q"], plain["s"], plain["w"], torch.ops.harp_block
    rows = harp_amd.Int8Rows(q, s)
    lin = harp_amd.Int8Linear(rows, w[:3])
    biased = harp_amd.Int8Linear(rows)
    biased.bias = dual(w[:3])
    qkv = (q.view(1, 3, 64), s.view(1, 3), [q.repeat(43, 1)[:128]], [s.repeat(43)[:128]])
    return [
        lambda: harp_amd.add_rms_norm(dual(f)), lambda: harp_amd.add_rms_norm(f, dual(f)),
        lambda: harp_amd.add_rms_norm(f, f, dual(w)),
        lambda: harp_amd.add_rms_norm(dual(f.clone().requires_grad_(True))),
        lambda: harp_amd.add_rms_norm_int8(dual(f)), lambda: harp_amd.add_rms_norm_int8(f, dual(f)),
        lambda: harp_amd.add_rms_norm_int8(f, None, dual(w)),
        lambda: harp_amd.quantize_int8(dual(f)), lambda: harp_amd.Int8Rows(q, dual(s)).dequantize(),
        lambda: harp_amd.int8_linear(harp_amd.Int8Rows(q, dual(s)), rows),
        lambda: harp_amd.int8_linear(rows, harp_amd.Int8Rows(q, dual(s))),
        lambda: harp_amd.int8_linear(rows, rows, dual(w[:3])),
        lambda: lin(dual(f)), lambda: lin(harp_amd.Int8Rows(q, dual(s))), lambda: biased(f), lambda: biased(rows),
        lambda: ops.qkv_int8(qkv[0], dual(qkv[1]), *qkv[2:], [None], [0.0], None),
        lambda: ops.qkv_int8(*qkv[:3], [dual(qkv[3][0])], [None], [0.0], None),
        lambda: ops.qkv_int8(*qkv, [dual(torch.ones_like(qkv[3][0]))], [1e-6], None),
    ]


def assert_tangents_are_refused(device):
    import torch.autograd.forward_ad as fwAD

    g = torch.Generator().manual_seed(1)
    plain = {"f": torch.randn(3, 64, generator=g), "s": torch.rand(3, generator=g), "w": torch.rand(64, generator=g),
             "q": torch.randint(-127, 128, (3, 64), generator=g, dtype=torch.int8)}
    plain = {k: v.to(device) for k, v in plain.items()}
    for grad in (True, False):
        with fwAD.dual_level(), torch.set_grad_enabled(grad):
            for i, call in enumerate(_dual_calls(lambda t: fwAD.make_dual(t, torch.ones_like(t)), plain)):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
                    pytest.fail(f"call {i} dropped its tangent")
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: harp_amd.quantize_int8(t)[1], (plain["f"],), (plain["f"],))


def test_forward_mode_derivatives_are_refused():
    assert_tangents_are_refused("cpu")


def test_operators_refuse_gradients():
    """The operators themselves, as the Python functions do."""
    ops = torch.ops.harp_block
    x, w = torch.zeros(3, 64, requires_grad=True), torch.zeros(64, requires_grad=True)
    q, s = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    ws = torch.zeros(3, requires_grad=True)
    for call in (lambda: ops.quantize_int8(x), lambda: ops.add_rms_norm_int8(x.detach(), None, w, 1e-5),
                 lambda: ops.linear_int8(q, s, q, ws, None, torch.float32),
                 lambda: ops.linear_int8_dynamic(x, q, s, None, torch.float32),
                 lambda: ops.dequantize_int8(q, ws, torch.float32),
                 lambda: ops.qkv_int8(q.view(1, 3, 64), s.view(1, 3), [q], [ws], [None], [0.0], None)):
        with pytest.raises(RuntimeError, match="forward only"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device only"):
            call()


@pytest.mark.parametrize("over,code,msg", [
    (dict(cols=2 ** 31 - 1, ldq=2 ** 31, ldo=2 ** 31), EUNSUPPORTED, "2^30"),  # 15 more would pass 31 bits
    (dict(cols=2 ** 30 + 1, ldq=2 ** 31, ldo=2 ** 31), EUNSUPPORTED, "2^30"),
    (dict(cols=0), EINVAL, "at least one value"),
    (dict(rows=-1), EINVAL, "at least one value"),
    (dict(q=FAKE + 8), EINVAL, "16-byte aligned"),
    (dict(ldq=48), EINVAL, "multiple of 16 in [64"),
    (dict(s=None), EINVAL, "scales is NULL"),
    (dict(o=None), EINVAL, "out is NULL"),
    (dict(ldo=63), EINVAL, "may not overlap"),
    (dict(od=2), EINVAL, "dtype"),
    (dict(rows=0, q=None), 0, ""),
])
def test_dequantize_refuses(over, code, msg):
    a = {**dict(q=FAKE, ldq=64, s=FAKE, o=FAKE, ldo=64, od=BF16, rows=4, cols=64), **over}
    rc = harp_amd.load_abi().harp_blk_dequantize_int8(a["q"], a["ldq"], a["s"], a["o"], a["ldo"], a["od"], a["rows"],
                                                      a["cols"], None)
    assert rc == code and msg in _err(), (rc, _err())


def test_every_kind_of_block_has_its_tests():
    """The shapes of the products' GPU tests run, on 256 CUs, in the kinds that the tests name, and reach every kind
    the library has, with a norm where the kind takes one, as the first launch of a call and as the second."""
    from tests.test_gpu_int8_linear import NORMED, PLAIN, product_plan

    _, _, kinds = product_plan(1, 1, 1, cus=256)
    plain, normed = {}, {}
    for M, N, K, want in PLAIN:
        launches, rows, _ = product_plan(M, N, K, cus=256)
        assert launches == want and (rows < M) == (len(want) == 2), (M, N, K, launches)
        for i, k in enumerate(launches):
            plain.setdefault(k, set()).add(i)
    for B, S, H, K, want in NORMED:
        launches, rows, _ = product_plan(B * S, 128 * H, K, 3, True, 256)
        assert launches == want and (rows < B * S) == (len(want) == 2), (B, S, H, K, launches)
        for i, k in enumerate(launches):
            normed.setdefault(k, set()).add(i)
    assert set(plain) == {k[:2] for k in kinds} and set(normed) == {k[:2] for k in kinds if k[2]}
    # every kind but the largest can be the second launch of a call
    largest = max(k[:2] for k in kinds)
    assert all(1 in plain[k[:2]] for k in kinds if k[:2] != largest)
    assert all(1 in normed[k[:2]] for k in kinds if k[2] and k[:2] != largest)


@pytest.mark.parametrize("name", ["to_q", "to_k", "to_v"])
def test_some_projections_in_8_bits_are_not_fused(name):
    """The fused bf16 kernel takes no module with an Int8Linear among its projections."""
    from harp_amd import qkv
    from tests.test_qk_abi import _DevView, _module

    attn, x = _module(), _DevView(torch.zeros(1, 16, 128, dtype=torch.bfloat16))
    assert qkv.fused_supported(attn, x, None)
    setattr(attn, name, harp_amd.Int8Linear(harp_amd.Int8Rows(torch.zeros(256, 128, dtype=torch.int8), torch.zeros(256))))
    assert not qkv.fused_supported(attn, x, None)
