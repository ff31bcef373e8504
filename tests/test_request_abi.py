"""CPU tests of the boundary of the operators for requests of one batch:
libharp_ra.so exports exactly the functions include/harp_request_ops.h declares,
bad arguments are refused on the host before any device call, and the Python
entry points refuse what they do not take (no GPU needed)."""

import ctypes
import math
import os
import re
import subprocess
from types import SimpleNamespace

import pytest
import torch
from torch import nn

import harp_amd
from harp_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "harp_request_ops.h")
FAKE = 1 << 20  # aligned, never dereferenced: validation fails first
EINVAL, EUNSUPPORTED, ENOMEM = 1, 2, 3
F32, BF16, I32, I64 = _lib.HARP_REQ_F32, _lib.HARP_REQ_BF16, _lib.HARP_REQ_I32, _lib.HARP_REQ_I64


def _err():
    return harp_amd.load_abi().harp_req_last_error().decode()


def test_header_prototypes_and_exports_agree():
    text = open(HEADER).read()
    fns = set(re.findall(r"HARP_REQ_API\s+[\w\s\*]+?\b(harp_req_\w+)\s*\(", text))
    assert fns == set(_lib.REQ_PROTOTYPES)
    nm = subprocess.run(["nm", "-D", "--defined-only", str(_lib.ABI_LIB)], capture_output=True, text=True)
    exported = {ln.split()[-1] for ln in nm.stdout.splitlines() if " T " in ln}
    assert {s for s in exported if s.startswith("harp_req_")} == fns


def test_structures_have_the_header_s_layout(tmp_path):
    """sizeof and the last member's offset of each structure, from a C compiler."""
    pairs = {"harp_req_axes_t": (_lib.ReqAxes, "half"), "harp_req_positions_t": (_lib.ReqPositions, "stride_a"),
             "harp_req_heads_t": (_lib.ReqHeads, "grad_weight"), "harp_req_requests_t": (_lib.ReqRequests, "count"),
             "harp_req_adapters_t": (_lib.ReqAdapters, "rank"), "harp_req_backward_set_t": (_lib.ReqBackwardSet, "db")}
    body = "".join(f'printf("%zu %zu\\n", sizeof({c}), offsetof({c}, {m}));' for c, (_, m) in pairs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{ {body} return 0; }}\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    for (t, m), line in zip(pairs.values(), lines):
        assert (ctypes.sizeof(t), getattr(t, m).offset) == tuple(int(v) for v in line.split())


def _axes(width=(32, 48, 48), theta=256.0, n=None, half=0):
    a = _lib.ReqAxes()
    a.half = half
    a.n = len(width) if n is None else n
    for i, w in enumerate(width):
        a.width[i], a.theta[i] = w, theta
    return a


def _positions(p=FAKE, dtype=I32):
    return _lib.ReqPositions(p, dtype, 0, 3, 1)


def _heads(H=2, D=128, **over):
    h = _lib.ReqHeads()
    h.x = h.y = h.dy = FAKE
    for name in ("x_stride", "y_stride", "dy_stride"):
        for i, v in enumerate((4 * H * D, D, H * D)):
            getattr(h, name)[i] = v
    h.heads, h.norm, h.weight, h.weight_dtype, h.eps = H, 1, FAKE, BF16, 1e-5
    for k, v in over.items():
        if k.endswith("stride"):
            for i, s in enumerate(v):
                getattr(h, k)[i] = s
        else:
            setattr(h, k, v)
    return h


def _rope(back=False, axes=None, pos=None, q=None, batch=1, seq=4, dtype=BF16, ws=FAKE, wsb=1 << 30):
    lib = harp_amd.load_abi()
    heads = (_lib.ReqHeads * 2)()
    heads[0] = _heads() if q is None else q
    axes, pos = _axes() if axes is None else axes, _positions() if pos is None else pos
    if back:
        return lib.harp_req_qk_norm_rope_backward(axes, pos, heads, batch, seq, dtype, ws, wsb, None)
    return lib.harp_req_qk_norm_rope_forward(axes, pos, heads, batch, seq, dtype, None)


ROPE = [
    (dict(axes=_axes(n=0)), EINVAL, "axes"),
    (dict(axes=_axes((2,) * 4, n=5)), EINVAL, "axes"),
    (dict(axes=_axes((3, 5))), EINVAL, "width[0]=3"),
    (dict(axes=_axes((2, 0))), EINVAL, "width[1]=0"),
    (dict(axes=_axes((128,), theta=0.0)), EINVAL, "theta"),
    (dict(axes=_axes((128,), theta=math.inf)), EINVAL, "theta"),
    (dict(axes=_axes((4, 2))), EUNSUPPORTED, "multiple of 8"),
    (dict(axes=_axes((256, 8))), EUNSUPPORTED, "at most 256"),
    (dict(pos=_positions(p=None)), EINVAL, "positions is NULL"),
    (dict(pos=_positions(dtype=BF16)), EINVAL, "positions dtype"),
    (dict(pos=_positions(p=FAKE + 4, dtype=I64)), EINVAL, "aligned"),
    (dict(batch=-1), EINVAL, "negative"),
    (dict(batch=1 << 20, seq=1 << 20), EUNSUPPORTED, "2^31"),
    (dict(dtype=I32), EINVAL, "dtype"),
    (dict(q=_heads(heads=-1)), EINVAL, "q.heads"),
    (dict(q=_heads(x=None)), EINVAL, "q.x"),
    (dict(q=_heads(x=FAKE + 8)), EINVAL, "q.x"),
    (dict(q=_heads(y=FAKE + 8)), EINVAL, "q.y"),
    (dict(q=_heads(x_stride=(1024, 128, 252))), EINVAL, "multiples of 8"),
    (dict(q=_heads(x_stride=(1024, 128, -256))), EINVAL, "not negative"),
    (dict(q=_heads(x_stride=(1024, 1 << 32, 256))), EINVAL, "below 2^31"),
    (dict(q=_heads(y_stride=(1024, 120, 256))), EINVAL, "one address"),
    (dict(q=_heads(y_stride=(1024, 128, 0))), EINVAL, "one address"),
    (dict(q=_heads(eps=-1.0)), EINVAL, "eps"),
    (dict(q=_heads(eps=math.nan)), EINVAL, "eps"),
    (dict(q=_heads(weight_dtype=I32)), EINVAL, "weight dtype"),
    (dict(q=_heads(weight=FAKE + 1)), EINVAL, "aligned"),
    (dict(q=_heads(norm=0)), EINVAL, "without a norm"),
]


@pytest.mark.parametrize("over,code,msg", ROPE)
@pytest.mark.parametrize("back", [False, True])
def test_rope_refuses(over, code, msg, back):
    rc = _rope(back, **over)
    assert rc == code and msg in _err(), (rc, _err())


@pytest.mark.parametrize("over,code,msg", [
    (dict(q=_heads(dy=None)), EINVAL, "q.dy"),
    (dict(q=_heads(grad_weight=FAKE, weight=None)), EINVAL, "grad_weight"),
    (dict(q=_heads(grad_weight=FAKE + 1)), EINVAL, "grad_weight"),
    (dict(q=_heads(grad_weight=FAKE), ws=None), ENOMEM, "workspace"),
    (dict(q=_heads(grad_weight=FAKE), wsb=8), ENOMEM, "workspace"),
    (dict(q=_heads(grad_weight=FAKE), ws=FAKE + 4), EINVAL, "workspace"),
])
def test_rope_backward_refuses(over, code, msg):
    rc = _rope(True, **over)
    assert rc == code and msg in _err(), (rc, _err())


def test_rope_does_nothing_without_tokens():
    assert harp_amd.load_abi().harp_req_qk_backward_workspace_bytes(1, 4, 128, 0, 0) == 0
    assert _rope(batch=0) == 0 and _rope(True, seq=0, ws=None, wsb=0) == 0 and _rope(q=_heads(heads=0)) == 0


def test_rope_workspace_and_table():
    lib = harp_amd.load_abi()
    size = lib.harp_req_qk_backward_workspace_bytes
    assert size(1, 8192, 128, 30, 30) % 512 == 0 and 0 < size(1, 8192, 128, 30, 30) <= 1024 * 128 * 4
    assert 0 < size(1, 1, 8, 1, 0) <= 64 and size(0, 5, 128, 3, 3) == 0
    for bad in ((-1, 1, 128, 1, 1), (1, 1, 12, 1, 1), (1, 1, 264, 1, 1), (1, 1, 128, -1, 1), (1 << 20, 1 << 11, 128, 1, 1)):
        assert size(*bad) == ctypes.c_size_t(-1).value
    rc = lib.harp_req_rope_table(_axes(), _positions(), 1, 4, None, None)
    assert rc == EINVAL and "table" in _err()
    rc = lib.harp_req_rope_table(_axes(), _positions(), 1, 4, FAKE + 4, None)
    assert rc == EINVAL and "table" in _err()
    assert lib.harp_req_rope_table(_axes(), None, 0, 4, None, None) == 0


ADD = dict(x=FAKE, ldx=64, base=FAKE, ldb=96, out=FAKE, ldo=96, dtype=BF16, a=FAKE, b=FAKE, s=None, n=2, rank=16,
           index=FAKE, idt=I32, offsets=FAKE, odt=I32, count=2, t=FAKE, T=6, K=64, N=96)


def _adapters(a):
    return (_lib.ReqAdapters(a["a"], a["b"], a["s"], a["n"], a["rank"]),
            _lib.ReqRequests(a["index"], a["idt"], a["offsets"], a["odt"], a["count"]))


def _add(**over):
    a = {**ADD, **over}
    ad, rq = _adapters(a)
    return harp_amd.load_abi().harp_req_add_adapters_forward(
        a["x"], a["ldx"], a["base"], a["ldb"], a["out"], a["ldo"], a["dtype"], ad, rq, a["t"], a["T"], a["K"], a["N"], None)


def _back(dy=FAKE, lddy=96, dx=FAKE, lddx=64, base=None, ldb=64, da=FAKE, db=FAKE, ws=FAKE, wsb=1 << 30, sets=1,
          second=None, **over):
    a = {**ADD, **over}
    ad, rq = _adapters(a)
    arr = (_lib.ReqBackwardSet * 3)()
    for i in range(3):
        arr[i] = _lib.ReqBackwardSet(ad, a["t"], dy, lddy, da, db)
    if second is not None:
        arr[1].adapters.rank = second
    return harp_amd.load_abi().harp_req_add_adapters_backward(
        arr if sets else None, sets, a["x"], a["ldx"], rq, base, ldb, dx, lddx, a["T"], a["K"], a["N"], ws, wsb, None)


BOTH = [
    (dict(T=-1), EINVAL, "tokens"),
    (dict(T=(1 << 25) + 1), EUNSUPPORTED, "2^25"),
    (dict(n=0), EINVAL, "n=0"),
    (dict(rank=0), EINVAL, "rank=0"),
    (dict(rank=129), EUNSUPPORTED, "rank=129"),
    (dict(n=(1 << 14) + 1), EUNSUPPORTED, "adapters"),
    (dict(K=0), EINVAL, "k_dim=0"),
    (dict(N=(1 << 22) + 1), EUNSUPPORTED, "2^22"),
    (dict(a=None), EINVAL, "a and b"),
    (dict(b=FAKE + 1), EINVAL, "a and b"),
    (dict(s=FAKE + 2), EINVAL, "scales"),
    (dict(index=None), EINVAL, "index is NULL"),
    (dict(idt=F32), EINVAL, "index dtype"),
    (dict(index=FAKE + 4, idt=I64), EINVAL, "index must be aligned"),
    (dict(odt=BF16), EINVAL, "offsets dtype"),
    (dict(offsets=FAKE + 2), EINVAL, "offsets must be aligned"),
    (dict(offsets=None, count=4), EINVAL, "one length"),
    (dict(count=0), EINVAL, "count=0"),
    (dict(count=(1 << 20) + 1), EUNSUPPORTED, "2^20"),
    (dict(x=None), EINVAL, "x is NULL"),
    (dict(x=FAKE + 1), EINVAL, "x must be aligned"),
    (dict(ldx=-1), EINVAL, "x row stride"),
    (dict(t=None), EINVAL, "t must be"),
    (dict(t=FAKE + 8), EINVAL, "t must be"),
]


@pytest.mark.parametrize("over,code,msg", BOTH)
@pytest.mark.parametrize("call", [_add, _back])
def test_adapters_refuse(over, code, msg, call):
    rc = call(**over)
    assert rc == code and msg in _err(), (rc, _err())


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=I32), EINVAL, "dtype"),
    (dict(base=None), EINVAL, "base is NULL"),
    (dict(out=None), EINVAL, "out is NULL"),
    (dict(out=FAKE + 64, ldo=95), EINVAL, "may not overlap"),
    (dict(dtype=F32, out=FAKE + 2), EINVAL, "out must be aligned"),
    (dict(ldo=128), EINVAL, "base's row stride"),
    (dict(ldb=0, ldo=0), EINVAL, "may not overlap"),
])
def test_adapters_forward_refuses(over, code, msg):
    rc = _add(**over)
    assert rc == code and msg in _err(), (rc, _err())


@pytest.mark.parametrize("over,code,msg", [
    (dict(dy=None), EINVAL, "dy is NULL"),
    (dict(lddy=-1), EINVAL, "dy row stride"),
    (dict(lddx=60), EINVAL, "may not overlap"),
    (dict(dx=FAKE + 1), EINVAL, "dx must be aligned"),
    (dict(da=FAKE + 1), EINVAL, "da and db"),
    (dict(ws=None), ENOMEM, "workspace"),
    (dict(wsb=64), ENOMEM, "workspace"),
    (dict(ws=FAKE + 8), EINVAL, "workspace"),
    (dict(sets=0), EINVAL, "1 to 3"),
    (dict(sets=4), EINVAL, "1 to 3"),
    (dict(sets=2, second=8), EINVAL, "sets[1]"),
    (dict(sets=3, rank=48), EINVAL, "dx_base"),
    (dict(base=FAKE + 2), EINVAL, "dx_base must be aligned"),
    (dict(base=FAKE, ldb=63), EINVAL, "dx_base row stride"),
])
def test_adapters_backward_refuses(over, code, msg):
    rc = _back(**over)
    assert rc == code and msg in _err(), (rc, _err())


def _qkv(x=FAKE, ldx=128, B=1, S=6, K=128, N=256, n_outs=3, ws=FAKE, wsb=1 << 30, t=None, adapters=True, odd=None,
         weight=FAKE, freqs=None, axes=None, pos=None, table=FAKE, **over):
    a = {**ADD, **over}
    ad, rq = _adapters(a)
    ads = (_lib.ReqAdapters * 3)(ad, ad, ad)
    if odd is not None:
        ads[2].rank = odd
    outs = (_lib.QkvOut * 3)()
    for o in outs:
        o.weight, o.ld_weight, o.y, o.ld_y = weight, K, FAKE, N
    ts = None if t is None else (ctypes.c_void_p * 3)(*[t] * 3)
    return harp_amd.load_abi().harp_req_qkv_project(x, ldx, B, S, K, N, freqs, 0, 128, axes, pos, table, outs,
                                                    ads if adapters else None, n_outs, rq, ts, ws, wsb, None)


@pytest.mark.parametrize("over,code,msg", [
    (dict(x=None), EINVAL, "x must be"),
    (dict(weight=FAKE + 8), EINVAL, "weight"),
    (dict(K=100), EUNSUPPORTED, "k_dim=100"),
    (dict(N=100), EUNSUPPORTED, "n_out=100"),
    (dict(n_outs=4), EINVAL, "1 to 3"),
    (dict(B=1 << 13, S=(1 << 12) + 1), EUNSUPPORTED, "2^25"),
    (dict(adapters=False), EINVAL, "adapters is NULL"),
    (dict(rank=0), EINVAL, "rank=0"),
    (dict(rank=12), EUNSUPPORTED, "multiple of 8"),
    (dict(b=FAKE + 8), EUNSUPPORTED, "16-byte"),
    (dict(odd=8), EINVAL, "adapters[2]"),
    (dict(index=None), EINVAL, "index is NULL"),
    (dict(offsets=None, count=4), EINVAL, "one length"),
    (dict(t=FAKE + 4), EINVAL, "t[0]"),
    (dict(axes=_axes(), pos=_positions(), freqs=FAKE), EINVAL, "one rotation"),
    (dict(axes=None, pos=_positions()), EINVAL, "axes is NULL"),
    (dict(axes=_axes((32, 32)), pos=_positions()), EUNSUPPORTED, "add up to 128"),
    (dict(axes=_axes(half=1), pos=_positions()), EUNSUPPORTED, "neighbouring pairs"),
    (dict(axes=_axes(), pos=_positions(dtype=BF16)), EINVAL, "positions dtype"),
    (dict(axes=_axes(), pos=_positions(), table=None), EINVAL, "table"),
    (dict(axes=_axes(), pos=_positions(), table=FAKE + 8), EINVAL, "table"),
    (dict(axes=_axes(), pos=_positions(), ws=None), ENOMEM, "workspace"),
    (dict(ws=None), ENOMEM, "workspace"),
    (dict(wsb=100), ENOMEM, "workspace"),
    (dict(ws=FAKE + 8), EINVAL, "workspace"),
])
def test_qkv_refuses(over, code, msg):
    rc = _qkv(**over)
    assert rc == code and msg in _err(), (rc, _err())
    size = harp_amd.load_abi().harp_req_qkv_workspace_bytes
    assert size(6, 16, 3) >= 3 * 6 * 64 and size(6, 0, 3) == size(6, 16, 4) == size(-1, 16, 1) == ctypes.c_size_t(-1).value


def test_adapters_sizes_and_empty_calls():
    lib = harp_amd.load_abi()
    assert [lib.harp_req_adapter_columns(r) for r in (1, 16, 17, 128)] == [16, 16, 32, 128]
    assert lib.harp_req_adapter_columns(0) == -1 and lib.harp_req_adapter_columns(129) == -1
    size = lib.harp_req_adapter_backward_workspace_bytes
    # u, and a and b transposed, at least
    assert size(6, 64, 96, 2, 16, 2, 1) >= 6 * 64 + 2 * 16 * (64 + 96) * 2
    for bad in ((-1, 64, 96, 2, 16, 2), (6, 0, 96, 2, 16, 2), (6, 64, 96, 0, 16, 2), (6, 64, 96, 2, 200, 2), (6, 64, 96, 2, 16, 0)):
        assert size(*bad, 1) == ctypes.c_size_t(-1).value
    assert size(6, 64, 96, 2, 16, 2, 0) == size(6, 64, 96, 2, 16, 2, 4) == ctypes.c_size_t(-1).value
    assert size(6, 64, 96, 2, 16, 2, 3) > size(6, 64, 96, 2, 16, 2, 1)
    assert _add(T=0, x=None, base=None, out=None, t=None) == 0 and _back(T=0, dy=None, ws=None, wsb=0) == 0
    assert _back(dx=None, da=None, db=None, ws=None, wsb=0) == 0


def test_python_refuses():
    for args, msg in [
        (((), 1.0), "one to 4 even"),
        (((2,) * 5, 1.0), "one to 4 even"),
        (((3,), 1.0), "even widths"),
        (((4, 4), (1.0,)), "theta"),
        (((4,), -1.0), "theta"),
        (((4,), math.nan), "theta"),
        (((4,), 1.0, "pairs"), "layout"),
    ]:
        with pytest.raises(ValueError, match=msg):
            harp_amd.AxialRope(*args)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    assert rope.dim == 128 and rope.theta == (256.0,) * 3 and "48" in repr(rope)
    q, p = torch.zeros(1, 2, 4, 128), torch.zeros(4, 3)
    for eps in (-1.0, (1e-5,), (1e-5, -1.0), math.nan):
        with pytest.raises(ValueError, match="eps"):
            harp_amd.qk_norm_axial_rope(q, None, p, rope, eps=eps)
    with pytest.raises(RuntimeError, match="HIP device only"):
        harp_amd.qk_norm_axial_rope(q, None, p, rope)
    with pytest.raises(RuntimeError, match="HIP device only"):
        harp_amd.AxialPositions(p, rope).table()
    low = harp_amd.Adapters(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4))
    with pytest.raises(RuntimeError, match="HIP device only"):
        harp_amd.add_adapters(torch.zeros(3, 6), torch.zeros(3, 8), low, harp_amd.AdapterRequests(torch.zeros(3)))


def test_modules_refuse():
    lin = nn.Linear(8, 6)
    A, L = harp_amd.Adapters, harp_amd.AdaptedLinear
    for low, msg in [(A(torch.zeros(2, 4, 7), torch.zeros(2, 6, 4)), "beside a weight"),
                     (A(torch.zeros(2, 4, 8), torch.zeros(2, 6, 3)), r"\[n, rank, in\]"),
                     (A(torch.zeros(4, 8), torch.zeros(6, 4)), r"\[n, rank, in\]"),
                     (A(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4), torch.ones(3)), "scales")]:
        with pytest.raises(ValueError, match=msg):
            L(lin, low)
    low = A(nn.Parameter(torch.zeros(2, 4, 8)), torch.zeros(2, 6, 4), torch.ones(2))
    m = L(lin, low)
    assert m.a is low.a and not m.b.requires_grad and m.b.data_ptr() == low.b.data_ptr()
    assert {n for n, _ in m.named_parameters()} == {"a", "b", "base.weight", "base.bias"}
    x = torch.randn(3, 8)
    assert torch.equal(m(x), lin(x))  # without requests the projection alone
    attn = SimpleNamespace(heads=1, to_q=lin, to_k=lin, to_v=lin)
    with pytest.raises(ValueError, match="to_out"):
        harp_amd.adapt_attention(attn, to_out=low)
    with pytest.raises(ValueError, match="adapt_attention"):
        harp_amd.project_qkv(attn, x, None, requests=harp_amd.AdapterRequests(torch.zeros(3)))


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.half().bfloat16(),
                                  lambda m: m.double().to("cpu", torch.bfloat16), lambda m: m.to("meta", torch.bfloat16)])
def test_scales_stay_float32_in_a_cast_module(cast):
    scales = torch.tensor([0.1, 1.7])  # (no bfloat16 values)
    lin = harp_amd.AdaptedLinear(nn.Linear(8, 6), harp_amd.Adapters(torch.zeros(2, 4, 8), torch.zeros(2, 6, 4), scales))
    m = cast(nn.Sequential(lin, harp_amd.AdaptedLinear(nn.Linear(6, 6), harp_amd.Adapters(torch.zeros(2, 4, 6), torch.zeros(2, 6, 4)))))
    assert all(p.dtype == torch.bfloat16 for p in m.parameters())
    assert m[0].scales.dtype == torch.float32 and m[0].scales.device == m[0].a.device and m[1].scales is None
    assert m[0].scales.is_meta or torch.equal(m[0].scales, scales)
    assert m[0]._buffers["scales"] is m[0].adapters.scales
