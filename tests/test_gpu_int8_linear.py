"""GPU tests of the products of 8-bit rows: harp_amd.int8_linear, Int8Linear
and the q/k/v producer on 8-bit projections, against the formulas in 64 bits.

Tolerances, with u = 2^-24 and half(t) half a step of the output's type: the
integer sums are exact, so y = acc a t + b carries one rounding of the sum's
conversion, two products and one addition:
|y - y64| <= 4 u (|acc a t| + |b|) + half |y64|.  A normed and rotated value
carries those, the norm's (64 squares a lane, a mean and a root: below 80 u),
and four more: 100 u (|a| + |b|) of its pair's sizes, and half a step."""

import pytest
import torch
from types import SimpleNamespace

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
B16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(g, rows, cols, pad=16, lead=0):
    """Random 8-bit rows, -127 .. 127, in storage whose padding holds other values."""
    ld = (lead + cols + pad - 1) // pad * pad
    store = torch.randint(-127, 128, (rows, ld), generator=g, dtype=torch.int8).to(DEV)
    scales = (torch.rand(rows, generator=g) * 0.02 + 1e-3).to(DEV)
    return harp_amd.Int8Rows(store[:, lead:lead + cols], scales)


def _exact(x, w):
    """The integer sums, exactly, in 64 bits."""
    return x.values.double() @ w.values.double().t()


def _assert_linear(y, x, w, bias, what):
    acc = _exact(x, w) * x.scales.double()[:, None] * w.scales.double()
    b = torch.zeros(w.values.size(0), device=DEV, dtype=torch.float64) if bias is None else bias.double()
    want = acc + b
    bound = 4 * U * (acc.abs() + b.abs()) + HALF[y.dtype] * want.abs()
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), (what, int((err > bound).sum()), float(err.max()))


MNK = [
    (1, 1, 1), (1, 16, 16), (1, 100, 64), (2, 128, 128), (5, 130, 129), (16, 256, 640), (17, 129, 1000), (31, 4, 33),
    (33, 300, 255), (64, 512, 512), (65, 513, 300), (127, 127, 127), (128, 128, 256), (129, 385, 384), (200, 1001, 70),
    (256, 256, 128), (257, 257, 257), (300, 96, 4097), (1000, 264, 512), (520, 1024, 48), (1, 3840, 3840),
    (3, 10240, 1000), (40, 17, 15360), (7, 33, 65536), (300, 2560, 640),
]


@pytest.mark.parametrize("M,N,K", MNK)
def test_linear(M, N, K):
    print(f"[int8_linear M={M} N={N} K={K}]", flush=True)
    g = _gen(M + 3 * N + 5 * K)
    x, w = _rows(g, M, K), _rows(g, N, K)
    for bias in (None, torch.randn(N, generator=g).to(B16).to(DEV), torch.randn(N, generator=g).to(DEV)):
        for dtype in (B16, F32):
            y = harp_amd.int8_linear(x, w, bias, dtype)
            assert y.shape == (M, N) and y.dtype == dtype and y.is_contiguous()
            _assert_linear(y, x, w, bias, (M, N, K, dtype))


def test_linear_layouts():
    """Rows out of wider storage, repeated rows, batches and vectors."""
    g = _gen(2)
    w = _rows(g, 200, 100, pad=64)
    x = _rows(g, 60, 100, pad=256, lead=48)
    _assert_linear(harp_amd.int8_linear(x, w), x, w, None, "wide rows")
    x1 = harp_amd.Int8Rows(x.values[:1].expand(40, 100), x.scales[:40].contiguous())
    _assert_linear(harp_amd.int8_linear(x1, w), x1, w, None, "repeated rows")
    xb = harp_amd.Int8Rows(x.values.unflatten(0, (3, 4, 5)), x.scales.view(3, 4, 5))
    assert torch.equal(harp_amd.int8_linear(xb, w).view(60, 200), harp_amd.int8_linear(x, w))
    xv = harp_amd.Int8Rows(x.values[7], x.scales[7])
    assert torch.equal(harp_amd.int8_linear(xv, w), harp_amd.int8_linear(x, w)[7])
    every = harp_amd.Int8Rows(x.values[::2], x.scales[::2])
    assert torch.equal(harp_amd.int8_linear(every, w), harp_amd.int8_linear(x, w)[::2])
    empty = harp_amd.Int8Rows(x.values[:0], x.scales[:0])
    assert harp_amd.int8_linear(empty, w).shape == (0, 200)


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_linear_extremes_and_nan(M):
    """The largest sums (K = 65536 of -127 * 127 and 127 * 127) are exact; a
    NaN scale makes its row NaN and no other."""
    K, N = 65536, 130
    x = torch.full((M, K), 127, dtype=torch.int8, device=DEV)
    w = torch.full((N, K), -127, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    s = torch.ones(M, device=DEV)
    t = torch.ones(N, device=DEV)
    y = harp_amd.int8_linear(harp_amd.Int8Rows(x, s), harp_amd.Int8Rows(w, t), None, F32)
    top = float(127 * 127 * K)  # 16129 * 2^16: exact in fp32
    assert bool((y[:, 1::2] == top).all()) and bool((y[:, 0::2] == -top).all())
    s[M // 2] = float("nan")
    y = harp_amd.int8_linear(harp_amd.Int8Rows(x, s), harp_amd.Int8Rows(w, t), None, F32)
    nan = torch.isnan(y).all(1)
    assert bool(nan[M // 2]) and int(nan.sum()) == 1 and int(torch.isnan(y).sum()) == N


def test_lowest_value():
    """-128, which no function here writes, multiplies as -128."""
    x = torch.full((40, 64), -128, dtype=torch.int8, device=DEV)
    one = torch.ones(40, device=DEV)
    y = harp_amd.int8_linear(harp_amd.Int8Rows(x, one), harp_amd.Int8Rows(x, one), None, F32)
    assert bool((y == 64 * 128 * 128).all())


@pytest.mark.parametrize("M", [1, 19, 333])
@pytest.mark.parametrize("dtype", [B16, F32], ids=str)
def test_module_quantises_its_input(M, dtype):
    g = _gen(M)
    lin = torch.nn.Linear(250, 321, bias=True)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(321, 250, generator=g) / 16)
        lin.bias.copy_(torch.randn(321, generator=g))
    lin = lin.to(B16).to(DEV)
    q = harp_amd.Int8Linear.from_linear(lin)
    x = torch.randn(2, M, 250, generator=g).to(dtype).to(DEV)
    rows = harp_amd.quantize_int8(x)
    y = q(x)
    assert y.shape == (2, M, 321) and torch.equal(y, q(rows))
    flat = harp_amd.Int8Rows(rows.values.view(2 * M, 250), rows.scales.view(-1))
    _assert_linear(y.view(2 * M, 321), flat, q.weight, lin.bias.detach(), "module")
    # and it stands in for the Linear: both operands are off by half a step of
    # max / 127 at most, a 250-term sum's error is within the sum of those
    full = x.double() @ lin.weight.detach().double().t() + lin.bias.detach().double()
    sx, sw = rows.scales.double(), q.weight.scales.double()
    bound = 0.5 * (sx[..., None] * q.weight.dequantize(F32).double().abs().sum(-1) + x.double().abs().sum(-1)[..., None] * sw) \
        + 250 * 0.25 * sx[..., None] * sw
    err = (y.double() - full).abs()
    assert bool((err <= 1.001 * bound + 2 ** -8 * full.abs()).all())


def test_linear_refusals():
    g = _gen(9)
    x, w = _rows(g, 4, 64), _rows(g, 32, 64)
    odd = torch.zeros(4, 70, dtype=torch.int8, device=DEV)[:, :64]
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        harp_amd.int8_linear(harp_amd.Int8Rows(odd, x.scales), w)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        harp_amd.int8_linear(harp_amd.Int8Rows(torch.zeros(4, 80, dtype=torch.int8, device=DEV)[:, 8:72], x.scales), w)
    with pytest.raises(RuntimeError, match="unit stride"):
        harp_amd.int8_linear(harp_amd.Int8Rows(torch.zeros(64, 4, dtype=torch.int8, device=DEV).t(), x.scales), w)
    with pytest.raises(RuntimeError, match="int8"):
        harp_amd.int8_linear(harp_amd.Int8Rows(x.values.float(), x.scales), w)
    with pytest.raises(RuntimeError, match="one scale for each row"):
        harp_amd.int8_linear(harp_amd.Int8Rows(x.values, x.scales[:3]), w)
    with pytest.raises(RuntimeError, match="float32"):
        harp_amd.int8_linear(harp_amd.Int8Rows(x.values, x.scales.to(B16)), w)
    with pytest.raises(RuntimeError, match=r"weight must be \[N, 64\]"):
        harp_amd.int8_linear(x, _rows(g, 32, 48))
    with pytest.raises(RuntimeError, match="bias"):
        harp_amd.int8_linear(x, w, torch.zeros(31, device=DEV))
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        harp_amd.int8_linear(x, w, None, torch.float16)


# ---------------------------------------------------------------------------
# q, k, v
# ---------------------------------------------------------------------------

def _freqs(S, batch=0):
    ang = torch.arange(S, dtype=torch.float64)[:, None] * (256.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128))
    if batch:
        ang = torch.stack([ang + 0.25 * b for b in range(batch)])
    return torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(DEV)


def _attn(g, H, K, norm_kind):
    to = [harp_amd.Int8Linear(_rows(g, H * 128, K)) for _ in range(3)]
    norms = [None, None]
    if norm_kind is not None:
        norms = [SimpleNamespace(weight=(1 + 0.2 * torch.randn(128, generator=g)).to(norm_kind).to(DEV), eps=1e-6)
                 for _ in range(2)]
    return SimpleNamespace(heads=H, to_q=to[0], to_k=to[1], to_v=to[2], norm_q=norms[0], norm_k=norms[1])


def _assert_qkv(outs, attn, rows, freqs, what):
    B, S = rows.scales.shape
    H = attn.heads
    flat = harp_amd.Int8Rows(rows.values.reshape(B * S, -1), rows.scales.reshape(-1))
    for i, (y, lin) in enumerate(zip(outs, (attn.to_q, attn.to_k, attn.to_v))):
        assert y.shape == (B, H, S, 128) and y.dtype == B16
        assert y.stride() == (S * H * 128, 128, H * 128, 1)
        want = (_exact(flat, lin.weight) * flat.scales.double()[:, None] * lin.weight.scales.double())
        want = want.view(B, S, H, 128).transpose(1, 2)
        norm = (attn.norm_q, attn.norm_k, None)[i]
        size, steps = want.abs(), 4
        if norm is not None:
            want = want / torch.sqrt(want.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
            size, steps = want.abs(), 100
            if freqs is not None:
                f = freqs.to(torch.complex128)
                f = f[:, None] if f.dim() == 3 else f
                pair = torch.view_as_complex(want.unflatten(-1, (64, 2)).contiguous())
                size = size.unflatten(-1, (64, 2)).sum(-1, keepdim=True).expand(*want.shape[:-1], 64, 2).flatten(-2)
                want = torch.view_as_real(pair * f).flatten(-2)
        err = (y.double() - want).abs()
        bound = steps * U * size + 2.0 ** -8 * want.abs()
        assert bool((err <= bound).all()), (what, i, int((err > bound).sum()), float(err.max()))


@pytest.mark.parametrize("B,S,H,K,norm,rope", [
    (1, 1, 1, 128, B16, True), (1, 1, 5, 640, F32, True), (2, 3, 2, 100, B16, False), (1, 40, 3, 384, B16, True),
    (2, 65, 2, 257, F32, True), (1, 128, 1, 128, None, False), (1, 300, 4, 512, B16, True), (3, 111, 3, 384, B16, True),
    (1, 700, 2, 1000, None, False), (1, 1030, 5, 640, F32, True),
    (1, 200, 30, 200, B16, True), (2, 350, 30, 130, F32, True), (2, 2100, 30, 100, B16, True), (5, 1333, 13, 64, B16, True), (1, 8100, 27, 1000, B16, True), (3, 2731, 28, 900, F32, True),
])
def test_qkv(B, S, H, K, norm, rope):
    print(f"[qkv B={B} S={S} H={H} K={K} norm={norm} rope={rope}]", flush=True)
    g = _gen(B + S + H + K)
    attn = _attn(g, H, K, norm)
    flat = _rows(g, B * S, K)
    rows = harp_amd.Int8Rows(flat.values.unflatten(0, (B, S)), flat.scales.view(B, S))
    freqs = _freqs(S, B if B > 2 else 0) if rope else None
    outs = harp_amd.project_qkv(attn, rows, freqs)
    _assert_qkv(outs, attn, rows, freqs, (B, S, H, K))


def test_qkv_unfused_paths():
    """What the one launch does not take runs as separate products and norms:
    the results agree to the bf16 steps between the stages (a product rounded
    to bf16, two values truncated to it: 2^-8 + 2 * 2^-7 of the pair, under
    2^-5 with the pair's other value)."""
    g = _gen(4)
    attn = _attn(g, 2, 256, B16)
    flat = _rows(g, 50, 256)
    rows = harp_amd.Int8Rows(flat.values.unflatten(0, (1, 50)), flat.scales.view(1, 50))
    f = _freqs(50)
    fused = harp_amd.project_qkv(attn, rows, f)
    apart = harp_amd.project_qkv(attn, rows, f, fused=False)
    for a, b in zip(fused, apart):
        assert a.shape == b.shape
        size = a.double().abs().unflatten(-1, (64, 2)).sum(-1, keepdim=True).expand(*a.shape[:-1], 64, 2).flatten(-2)
        assert bool(((a.double() - b.double()).abs() <= 2 ** -5 * size + 1e-6).all())
    assert torch.equal(fused[2], apart[2])
    # a bias keeps the products apart
    attn.to_v = harp_amd.Int8Linear(attn.to_v.weight, torch.ones(256, device=DEV))
    v = harp_amd.project_qkv(attn, rows, f)[2]
    assert torch.equal(v, attn.to_v(rows).unflatten(-1, (2, 128)).transpose(1, 2))


@pytest.mark.parametrize("M,N", [(1, 2 ** 28 + 40), (2 ** 27 + 9, 3)])
def test_more_blocks_than_one_launch_holds(M, N):
    """A grid holds fewer than 2^32 threads: the smallest blocks make way."""
    K = 16
    g = torch.Generator(DEV).manual_seed(M % 97)
    x, w = (harp_amd.Int8Rows(torch.empty(n, K, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g),
                              torch.rand(n, generator=g, device=DEV)) for n in (M, N))
    y = harp_amd.int8_linear(x, w)
    for lo in (0, max(M, N) // 2, max(M, N) - 512):
        s = slice(lo, lo + 512)
        if M == 1:
            _assert_linear(y[:, s], x, harp_amd.Int8Rows(w.values[s], w.scales[s]), None, lo)
        else:
            _assert_linear(y[s], harp_amd.Int8Rows(x.values[s], x.scales[s]), w, None, lo)


def test_weight_of_other_width_is_refused():
    x = harp_amd.quantize_int8(torch.ones(3, 40, device=DEV))
    for cols in (64, 47, 32):
        w = harp_amd.quantize_int8(torch.ones(8, cols, device=DEV))
        with pytest.raises(RuntimeError, match="weight must be"):
            torch.ops.harp_block.linear_int8(x.values, x.scales, w.values, w.scales, None, B16)


@pytest.mark.parametrize("K", [1008, 1024, 1030, 2570])
def test_module_with_padded_rows(K):
    """Long weight rows are padded to whole cache lines: same results as unpadded ones."""
    g = _gen(K)
    w = _rows(g, 200, K, pad=16)
    lin = harp_amd.Int8Linear(w)
    assert lin.weight_values.size(1) == (1008 if K == 1008 else -(-K // 128) * 128)
    assert torch.equal(lin.weight.values, w.values) and bool((lin.weight_values[:, K:] == 0).all())
    for M in (1, 20, 150):
        x = _rows(g, M, K)
        y = lin(x)
        assert torch.equal(y, harp_amd.int8_linear(x, w))
        _assert_linear(y, x, w, None, M)
        xf = torch.randn(M, K, generator=g).to(DEV)
        assert torch.equal(lin(xf), lin(harp_amd.quantize_int8(xf)))


@pytest.mark.parametrize("K,wide", [(40, 48), (40, 56), (1001, 1024), (2570, 2576), (2570, 2688)])
def test_wider_weight_is_refused(K, wide):
    """Columns are dropped only where in_features says how many count."""
    harp_amd.load_block_ops()
    ops = torch.ops.harp_block
    g = _gen(K)
    x, w = _rows(g, 3, K), _rows(g, 8, wide)
    xf = torch.randn(3, K, generator=g).to(DEV)
    for call in (lambda: ops.linear_int8(x.values, x.scales, w.values, w.scales, None, F32),
                 lambda: ops.linear_int8_dynamic(xf, w.values, w.scales, None, F32),
                 lambda: ops.linear_int8(x.values, x.scales, w.values, w.scales, None, F32, K - 1),
                 lambda: ops.linear_int8(x.values, x.scales, w.values, w.scales, None, F32, wide),
                 lambda: ops.linear_int8(x.values, x.scales, w.values[:, :K - 1], w.scales, None, F32, K)):
        with pytest.raises(RuntimeError, match="must (be|have)"):
            call()
    first = harp_amd.Int8Rows(w.values[:, :K], w.scales)
    y = ops.linear_int8(x.values, x.scales, w.values, w.scales, None, F32, K)
    assert torch.equal(y, harp_amd.int8_linear(x, first, None, F32))
    _assert_linear(y, x, first, None, (K, wide))


# ---------------------------------------------------------------------------
# every kind of block
# ---------------------------------------------------------------------------

def product_plan(M, N, K, n_outs=1, norm=False, cus=0):
    """((tokens, features) of the blocks of a product's one or two launches, the first one's rows, all kinds)."""
    import ctypes

    out, kinds = (ctypes.c_int * 5)(), (ctypes.c_int * 96)()
    n = harp_amd.load_abi().harp_prod8_plan(M, N, K, n_outs, int(norm), cus, out, kinds, 32)
    assert 0 < n <= 32
    launches = [(out[0], out[1])] + ([(out[3], out[4])] if out[3] else [])
    return launches, out[2], [tuple(kinds[3 * i:3 * i + 3]) for i in range(n)]


# tokens, features, K (none a multiple of 16) and the launches that such a product runs as on 256 CUs
PLAIN = [
    (9, 41, 5483, [(16, 16)]),
    (540, 37, 3123, [(32, 32)]),
    (269, 1533, 1971, [(32, 64)]),
    (91, 8771, 3571, [(32, 128)]),
    (422, 5643, 571, [(64, 64)]),
    (265, 5251, 3215, [(64, 128)]),
    (558, 5545, 1817, [(128, 128)]),
    (2834, 2365, 1515, [(128, 256)]),
    (2184, 4413, 2195, [(256, 256)]),
    (905, 4207, 5363, [(128, 128), (16, 16)]),
    (1415, 5405, 2331, [(128, 256), (32, 32)]),
    (1195, 6985, 2561, [(128, 256), (32, 64)]),
    (2718, 3279, 5603, [(128, 256), (32, 128)]),
    (1236, 7079, 2721, [(128, 256), (64, 64)]),
    (1179, 8089, 4707, [(128, 256), (64, 128)]),
    (3378, 5727, 1541, [(256, 256), (128, 128)]),
    (2367, 8847, 1485, [(256, 256), (128, 256)]),
]
# batch, tokens, heads, K of a q/k/v product with norms
NORMED = [
    (1, 271, 2, 555, [(32, 128)]),
    (1, 361, 8, 2265, [(64, 128)]),
    (2, 258, 14, 1845, [(128, 128)]),
    (1, 900, 15, 2055, [(128, 256)]),
    (1, 1372, 27, 2121, [(256, 256)]),
    (2, 326, 29, 4209, [(128, 256), (32, 128)]),
    (1, 932, 28, 4281, [(128, 256), (64, 128)]),
    (1, 2390, 17, 3215, [(256, 256), (32, 128)]),
    (2, 1262, 17, 2531, [(256, 256), (64, 128)]),
    (3, 1015, 16, 2509, [(256, 256), (128, 128)]),
    (1, 3337, 29, 1463, [(256, 256), (128, 256)]),
]


@pytest.mark.parametrize("M,N,K,kinds", PLAIN)
def test_linear_in_every_kind_of_block(M, N, K, kinds):
    """Tails in all three sizes over several K-tiles, both result types and all biases; every result within bounds
    and the same as in a call of some of the rows."""
    print(f"[int8_linear M={M} N={N} K={K} {kinds}]", flush=True)
    launches, rows, _ = product_plan(M, N, K)
    assert launches == kinds
    g = _gen(M + N)
    x, w = _rows(g, M, K), _rows(g, N, K)
    acc = _exact(x, w) * x.scales.double()[:, None] * w.scales.double()
    some = harp_amd.Int8Rows(x.values[max(0, rows - 9):rows + 7], x.scales[max(0, rows - 9):rows + 7])
    for bias in (None, torch.randn(N, generator=g).to(B16).to(DEV), torch.randn(N, generator=g).to(DEV)):
        b = torch.zeros(N, device=DEV, dtype=torch.float64) if bias is None else bias.double()
        for dtype in (B16, F32):
            y = harp_amd.int8_linear(x, w, bias, dtype)
            want = acc + b
            err = (y.double() - want).abs()
            bad = err > 4 * U * (acc.abs() + b.abs()) + HALF[dtype] * want.abs()
            assert not bool(bad.any()), (dtype, int(bad.sum()), bad.nonzero()[0].tolist(), float(err.max()))
            assert torch.equal(harp_amd.int8_linear(some, w, bias, dtype), y[max(0, rows - 9):rows + 7])


@pytest.mark.parametrize("M,N,K", [(8000, 5001, 100), (8000, 3841, 1), (1000, 5000, 100), (600, 8000, 100), (2049, 2049, 127),
                                   (4100, 4100, 127), (8000, 3000, 257)])
def test_linear_of_few_k_tiles(M, N, K):
    print(f"[int8_linear M={M} N={N} K={K} {product_plan(M, N, K)[0]}]", flush=True)
    g = _gen(M + K)
    x, w = _rows(g, M, K), _rows(g, N, K)
    bias = torch.randn(N, generator=g).to(DEV)
    for dtype in (B16, F32):
        _assert_linear(harp_amd.int8_linear(x, w, bias, dtype), x, w, bias, (M, N, K, dtype))


@pytest.mark.parametrize("B,S,H,K,kinds", NORMED)
@pytest.mark.parametrize("norm", [B16, F32], ids=str)
def test_qkv_in_every_kind_of_block(B, S, H, K, kinds, norm):
    print(f"[qkv B={B} S={S} H={H} K={K} norm={norm} {kinds}]", flush=True)
    assert product_plan(B * S, 128 * H, K, 3, True)[0] == kinds
    g = _gen(B + S + H + K)
    attn = _attn(g, H, K, norm)
    flat = _rows(g, B * S, K)
    rows = harp_amd.Int8Rows(flat.values.unflatten(0, (B, S)), flat.scales.view(B, S))
    freqs = _freqs(S, B if B > 1 else 0) if norm == B16 else None
    _assert_qkv(harp_amd.project_qkv(attn, rows, freqs), attn, rows, freqs, (B, S, H, K))
    if norm == F32:
        return
    attn.norm_q = attn.norm_k = None  # the same sizes without a norm run in other kinds
    _assert_qkv(harp_amd.project_qkv(attn, rows, None), attn, rows, None, (B, S, H, K))


@pytest.mark.parametrize("B,S,H,K,kinds", [c for c in NORMED if c[0] == 1])
def test_qkv_does_not_depend_on_the_batch(B, S, H, K, kinds):
    """A token's q, k and v are the same alone, among a few and among all, whatever kinds of blocks the calls run in."""
    g = _gen(S)
    attn, flat, freqs = _attn(g, H, K, B16), _rows(g, S, K), _freqs(S)
    full = harp_amd.project_qkv(attn, harp_amd.Int8Rows(flat.values[None], flat.scales[None]), freqs)
    seen = {tuple(kinds)}
    for n in (1, 40, 70, 200, 300, 520):
        n = min(n, S)
        seen.add(tuple(product_plan(n, 128 * H, K, 3, True)[0]))
        for s in (slice(0, n), slice(S - n, S)):
            some = harp_amd.project_qkv(attn, harp_amd.Int8Rows(flat.values[None, s], flat.scales[None, s]), freqs[s])
            for name, a, b in zip("qkv", full, some):
                assert torch.equal(a[:, :, s], b), (name, n, int((a[:, :, s] != b).sum()))
    assert len(seen) > 1 or H * K < 5000, seen


def test_rope_table_forms():
    """The complex table and its (cos, sin) rows give the same; view_as_real's own shape is refused with what is taken."""
    g = _gen(3)
    attn, flat, f = _attn(g, 2, 256, B16), _rows(g, 30, 256), _freqs(30)
    rows = harp_amd.Int8Rows(flat.values[None], flat.scales[None])
    want = harp_amd.project_qkv(attn, rows, f)
    got = harp_amd.project_qkv(attn, rows, torch.view_as_real(f).flatten(-2))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for bad in (torch.view_as_real(f), f[:29], f.to(torch.complex128)):
        with pytest.raises(RuntimeError, match=r"float32 \(cos, sin\) rows \[\.\., S, 128\]"):
            harp_amd.project_qkv(attn, rows, bad)
