"""GPU tests of the residual addition with its RMSNorm (harp_amd.add_rms_norm,
add_rms_norm_int8) and of 8-bit rows (quantize_int8, Int8Rows.dequantize),
against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and half(t) half a step of the
output's type (2^-8 for bf16, u for fp32):
* h is the fp32 sum rounded to its type: equal bit for bit.
* The sum of squares has at most 64 values per thread and 10 exchange steps in
  sequence, so rho = 1 / rms carries at most (74 / 2 + 4) u, y three more
  products: |y - y64| <= (half + 64 u) |y64|.
* dx = rho (g - n c) + dh with c = mean(g n): each factor carries at most 64 u
  of its own size and c at most 64 u of mean |g n|, five operations follow:
  192 u (rho (|g| + |n| mean |g n|) + |dh|) + half |dx64|.
* dw sums T products, in blocks: (T + 64) u sum |dy n| + half |dw64|.
* quantize_int8 is exact: equal to round(127 x / max) in 64 bits, and the scale
  one division off (u).
* The 8-bit rows of the norm: the quotient 127 h w / max |h w| carries at most
  5 u of at most 127, so a value may differ by one step only where the 64-bit
  quotient lies that close to a border; the scale carries 64 u."""

import pytest
import torch

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
B16, F32 = torch.bfloat16, torch.float32


def _rand(g, *shape, dtype=B16, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _assert_within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = err > bound
    assert not bool(bad.any()), (what, int(bad.sum()), float((err - bound).max()), float(err.max()))


SHAPES = [  # rows, cols
    (1, 1), (1, 64), (3, 7), (5, 8), (2, 129), (17, 513), (64, 512), (9, 1023), (33, 1025), (7, 2048), (300, 3840),
    (11, 3841), (4, 8191), (3, 10240), (2, 16385), (3, 32768), (1100, 200),
]
TYPES = [  # x, residual, weight
    (B16, B16, B16), (B16, F32, F32), (F32, B16, None), (F32, F32, B16), (B16, None, B16), (F32, None, F32),
]


def _case(rows, cols, types, seed):
    xd, rd, wd = types
    g = _gen(seed)
    x = _rand(g, rows, cols, dtype=xd)
    r = None if rd is None else _rand(g, rows, cols, dtype=rd, scale=2.0)
    w = None if wd is None else (1 + _rand(g, cols, dtype=F32, scale=0.2)).to(wd)
    return g, x, r, w


def _norm64(h, w, eps):
    hd = h.double()
    rho = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    n = hd * rho
    return n if w is None else n * w.double(), n, rho


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_backward(rows, cols, types):
    print(f"[add_rms_norm rows={rows} cols={cols} types={types}]", flush=True)
    g, x, r, w = _case(rows, cols, types, rows * 7 + cols)
    eps = 1e-5
    for t in (x, r, w):
        if t is not None:
            t.requires_grad_(True)
    y, h = harp_amd.add_rms_norm(x, r, w, eps)
    dy = _rand(g, rows, cols, dtype=x.dtype)
    want_h = x if r is None else (x.detach().float() + r.detach().float()).to(r.dtype)
    assert h.dtype == want_h.dtype and torch.equal(h, want_h)
    y64, n64, rho64 = _norm64(want_h.detach(), None if w is None else w.detach(), eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    _assert_within(y, y64, (HALF[x.dtype] + 64 * U) * y64.abs(), "y")

    dh = _rand(g, rows, cols, dtype=h.dtype) if r is not None else None
    leaves = [t for t in (x, r, w) if t is not None]
    outs, grads = ((y, h), (dy, dh)) if r is not None else ((y,), (dy,))
    got = list(torch.autograd.grad(outs, leaves, grads))
    gw64 = dy.double() if w is None else dy.double() * w.detach().double()
    mean_abs = (gw64 * n64).abs().mean(-1, keepdim=True)
    dx64 = rho64 * (gw64 - n64 * (gw64 * n64).mean(-1, keepdim=True))
    size = rho64 * (gw64.abs() + n64.abs() * mean_abs)
    if dh is not None:
        dx64, size = dx64 + dh.double(), size + dh.double().abs()
    for t, name in ((x, "dx"), (r, "dresidual")):
        if t is not None:
            d = got.pop(0)
            assert d.dtype == t.dtype and d.shape == t.shape
            _assert_within(d, dx64, 192 * U * size + HALF[t.dtype] * dx64.abs(), name)
    if w is not None:
        d = got.pop(0)
        assert d.dtype == w.dtype
        dn = dy.double() * n64
        _assert_within(d, dn.sum(0), (rows + 64) * U * dn.abs().sum(0) + HALF[w.dtype] * dn.sum(0).abs(), "dweight")


def test_gradient_against_differences():
    """The directional derivative of sum(y a) + sum(h b) in fp32 against
    central differences of the 64-bit forward.  The differences' own error is
    of order step^2 times the third derivative (step 1e-4: below 1e-6
    relative); the gradient's is below 1e-4 of the terms that it sums."""
    g = _gen(5)
    x, r, w = _rand(g, 6, 40, dtype=F32), _rand(g, 6, 40, dtype=F32), 1 + _rand(g, 40, dtype=F32, scale=0.2)
    a, b = _rand(g, 6, 40, dtype=F32), _rand(g, 6, 40, dtype=F32)
    dirs = [_rand(g, *t.shape, dtype=F32) for t in (x, r, w)]

    def value(s):
        xs, rs, ws = (t.double() + s * d.double() for t, d in zip((x, r, w), dirs))
        y, _, _ = _norm64(xs + rs, ws, 1e-5)
        return float((y * a.double()).sum() + ((xs + rs) * b.double()).sum())

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = harp_amd.add_rms_norm(*leaves, 1e-5)
    grads = torch.autograd.grad((y, h), leaves, (a, b))
    got = sum(float((gr.double() * d.double()).sum()) for gr, d in zip(grads, dirs))
    size = sum(float((gr.double() * d.double()).abs().sum()) for gr, d in zip(grads, dirs))
    want = (value(1e-4) - value(-1e-4)) / 2e-4
    assert abs(got - want) <= 1e-5 * size, (got, want, size)


def test_unused_outputs():
    """Gradients where only y, or only h, takes part."""
    g, x, r, w = _case(5, 96, (B16, F32, B16), 3)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, h = harp_amd.add_rms_norm(x, r, w)
    d = _rand(g, 5, 96, dtype=F32)
    gx, gr, gw = torch.autograd.grad(h, (x, r, w), d, retain_graph=True, allow_unused=True)
    assert torch.equal(gx, d.to(B16)) and torch.equal(gr, d) and gw is None
    dy = _rand(g, 5, 96)
    zero = torch.zeros_like(h)
    both = torch.autograd.grad((y, h), (x, r, w), (dy, zero), retain_graph=True)
    only = torch.autograd.grad(y, (x, r, w), dy)
    assert all(torch.equal(p, q) for p, q in zip(both, only))


@pytest.mark.parametrize("xd,rd", [(B16, B16), (B16, F32), (F32, None)], ids=str)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm_int8(rows, cols, xd, rd):
    print(f"[add_rms_norm_int8 rows={rows} cols={cols} {xd} {rd}]", flush=True)
    g, x, r, w = _case(rows, cols, (xd, rd, B16), rows + cols)
    (q, s), h = harp_amd.add_rms_norm_int8(x, r, w, 1e-5)
    want_h = x if r is None else (x.float() + r.float()).to(r.dtype)
    assert torch.equal(h, want_h)
    y64, _, _ = _norm64(want_h, w, 1e-5)
    most = y64.abs().amax(-1, keepdim=True)
    t64 = 127 * y64 / most
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == x.shape[:-1] and q.stride(-1) == 1
    _assert_within(s, (most / 127).squeeze(-1), 64 * U * (most / 127).squeeze(-1), "scale")
    off = (q.double() - t64.round()).abs()
    near = ((t64 - t64.floor() - 0.5).abs() <= 127 * 5 * U).double()
    assert bool((off <= near).all()), int((off > near).sum())
    # the bytes that pad the rows are zeros
    full = q.as_strided((rows, q.stride(0) if rows > 1 else -(-cols // 16) * 16), (q.stride(0), 1))
    assert bool((full[:, cols:] == 0).all())


@pytest.mark.parametrize("dtype", [B16, F32], ids=str)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_is_exact(rows, cols, dtype):
    print(f"[quantize_int8 rows={rows} cols={cols} {dtype}]", flush=True)
    x = _rand(_gen(cols), rows, cols, dtype=dtype)
    x[0, : cols // 2] = x[0].abs().max() / 2  # halfway between two steps: to the even one
    q, s = harp_amd.quantize_int8(x)
    most = x.double().abs().amax(-1, keepdim=True)
    assert torch.equal(q.double(), torch.round(127 * x.double() / most))
    _assert_within(s, most.squeeze(-1) / 127, U * most.squeeze(-1) / 127, "scale")
    for out in (B16, F32):
        v = harp_amd.Int8Rows(q, s).dequantize(out)
        assert v.dtype == out and torch.equal(v, (q.float() * s[:, None]).to(out))


def test_quantize_special_rows():
    """Zeros, the smallest and largest values, infinities and NaN."""
    x = torch.zeros(9, 40)
    x[1] = 2.0 ** -149 * torch.arange(40)               # fp32 denormals: the maximum 39 steps of 2^-149
    x[2] = 2.0 ** -120 * torch.linspace(-1, 1, 40)
    x[3] = 3.0e38 * torch.linspace(-1, 1, 40)
    x[4, 3] = float("inf")
    x[5, 39] = float("-inf")
    x[6, 0] = float("nan")
    x[7, 5] = -4.0                                      # one value: -127
    x[8] = 1.0
    x = x.to(DEV)
    q, s = harp_amd.quantize_int8(x)
    assert bool((q[0] == 0).all()) and float(s[0]) == 0.0
    for i in (1, 2, 3, 8):
        most = x[i].double().abs().max()
        assert torch.equal(q[i].double(), torch.round(127 * x[i].double() / most)), i
    assert abs(float(s[2]) - 2.0 ** -120 / 127) <= U * 2.0 ** -120 / 127
    # a denormal scale is rounded to the denormals' step
    assert abs(float(s[1]) - 39 * 2.0 ** -149 / 127) <= 2.0 ** -150
    for i in (4, 5, 6):
        assert bool((q[i] == 0).all()) and bool(torch.isnan(s[i])), i
    assert int(q[7, 5]) == -127 and int(q[7].abs().sum()) == 127
    assert bool(torch.isnan(harp_amd.Int8Rows(q, s).dequantize()[4]).all())


def test_norm_special_rows():
    """A padding row of zeros gives zeros (and finite gradients); an infinity
    or a NaN stays in its row."""
    x = torch.randn(5, 72).to(B16)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x = x.to(DEV).requires_grad_(True)
    w = torch.ones(72, device=DEV)
    y, _ = harp_amd.add_rms_norm(x, None, w)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool((y[1] == 0).all()) and bool(torch.isfinite(dx[1]).all())
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[2, 7]))
    for i in (0, 4):
        assert bool(torch.isfinite(y[i]).all()) and bool(torch.isfinite(dx[i]).all())
    rows, _ = harp_amd.add_rms_norm_int8(x.detach(), None, w)
    assert bool((rows.values[1] == 0).all()) and float(rows.scales[1]) == 0.0
    assert bool(torch.isnan(rows.scales[2:4]).all()) and bool((rows.values[2:4] == 0).all())
    assert bool(torch.isfinite(rows.scales[[0, 1, 4]]).all())


def test_strided_inputs_and_shapes():
    """Row strides, unaligned rows, higher ranks, expanded and transposed
    inputs give what their contiguous copies give, bit for bit."""
    g = _gen(11)
    wide = _rand(g, 6, 5, 301)
    w = _rand(g, 200, dtype=F32)
    views = [wide[:, :, 50:250], wide[:, :, 1:201], wide[:, 2, 3:203], wide[::2, 1:4, :200],
             wide[:1, :1, :200].expand(6, 5, 200), _rand(g, 200, 6, 5).permute(2, 1, 0), wide[0, 0, :200]]
    for i, v in enumerate(views):
        print(f"[view {i}: {tuple(v.shape)} {v.stride()}]", flush=True)
        r = _rand(g, *v.shape)
        y, h = harp_amd.add_rms_norm(v, r, w)
        y2, h2 = harp_amd.add_rms_norm(v.contiguous(), r, w)
        assert y.shape == v.shape and torch.equal(y, y2) and torch.equal(h, h2)
        y, h = harp_amd.add_rms_norm(r, v, w)
        y2, h2 = harp_amd.add_rms_norm(r, v.contiguous(), w)
        assert torch.equal(y, y2) and torch.equal(h, h2)
        a, b = harp_amd.quantize_int8(v), harp_amd.quantize_int8(v.contiguous())
        assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)
    # gradients of an expanded input, and with an expanded gradient
    x1, r = wide[:1, :1, :200].clone().requires_grad_(True), _rand(g, 6, 5, 200).requires_grad_(True)
    y, h = harp_amd.add_rms_norm(x1.expand(6, 5, 200), r, w)
    one = torch.ones(1, 1, 1, device=DEV, dtype=B16).expand(6, 5, 200)
    gx, gr = torch.autograd.grad((y, h), (x1, r), (one, one))
    x2 = x1.detach().expand(6, 5, 200).contiguous().requires_grad_(True)
    y2, h2 = harp_amd.add_rms_norm(x2, r, w)
    gx2, gr2 = torch.autograd.grad((y2, h2), (x2, r), (one.contiguous(), one.contiguous()))
    assert torch.equal(gr, gr2) and gx.shape == x1.shape
    torch.testing.assert_close(gx, gx2.float().sum((0, 1), keepdim=True).to(B16), rtol=2 ** -7, atol=0.05)


def test_empty_batches():
    x = torch.empty(0, 64, device=DEV, dtype=B16).requires_grad_(True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, h = harp_amd.add_rms_norm(x, x.detach(), w)
    gx, gw = torch.autograd.grad((y, h), (x, w), (y.detach(), h.detach()))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and bool((gw == 0).all())
    rows, _ = harp_amd.add_rms_norm_int8(x.detach(), None, w.detach())
    assert rows.values.shape == (0, 64) and rows.scales.shape == (0,)
    assert harp_amd.quantize_int8(x.detach()).dequantize().shape == (0, 64)


def test_refusals():
    x = torch.zeros(3, 64, device=DEV, dtype=B16)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        harp_amd.add_rms_norm(x.half())
    with pytest.raises(RuntimeError, match="shape"):
        harp_amd.add_rms_norm(x, x[:1])
    with pytest.raises(RuntimeError, match="weight must be a vector of 64"):
        harp_amd.add_rms_norm(x, None, torch.ones(63, device=DEV))
    with pytest.raises(RuntimeError, match="device"):
        harp_amd.add_rms_norm(x, x.cpu())
    with pytest.raises(RuntimeError, match="eps"):
        harp_amd.add_rms_norm(x, None, None, -1.0)
    with pytest.raises(RuntimeError, match="32768"):
        harp_amd.quantize_int8(torch.zeros(1, 32769, device=DEV))
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        harp_amd.quantize_int8(x).dequantize(torch.float16)


def test_outputs_next_to_others_are_left_alone():
    """The C entry points write cols columns of rows rows: what lies between
    and behind the rows of a padded output stays as it was (the 8-bit rows are
    written up to the next multiple of 16)."""
    import ctypes

    from harp_amd import _lib

    lib = harp_amd.load_abi()
    rows, cols, ld = 5, 77, 96
    g = _gen(1)
    x, r = _rand(g, rows, cols), _rand(g, rows, cols)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    y, h = (torch.full((rows + 2, ld), 7.0, device=DEV, dtype=B16) for _ in range(2))
    rc = lib.harp_blk_add_rms_norm_forward(x.data_ptr(), cols, 1, r.data_ptr(), cols, 1, None, 1, 1e-5, y.data_ptr(),
                                           ld, h.data_ptr(), ld, None, rows, cols, stream)
    assert rc == 0
    want_y, want_h = harp_amd.add_rms_norm(x, r)
    for t, want in ((y, want_y), (h, want_h)):
        assert torch.equal(t[:rows, :cols], want)
        assert bool((t[:rows, cols:] == 7).all()) and bool((t[rows:] == 7).all())
    q = torch.full((rows + 2, ld), 9, device=DEV, dtype=torch.int8)
    s = torch.empty(rows, device=DEV)
    rc = lib.harp_blk_quantize_int8(x.data_ptr(), cols, 1, q.data_ptr(), ld, s.data_ptr(), rows, cols, stream)
    assert rc == 0
    assert torch.equal(q[:rows, :cols], harp_amd.quantize_int8(x).values)
    assert bool((q[:rows, cols:80] == 0).all()) and bool((q[:rows, 80:] == 9).all()) and bool((q[rows:] == 9).all())


def test_differentiable_once():
    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    y, _ = harp_amd.add_rms_norm(x)
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        gx.sum().backward()


def test_saved_tensors_are_guarded():
    """h is kept for the backward: changing it in place raises there."""
    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    y, h = harp_amd.add_rms_norm(x, torch.zeros(3, 64, device=DEV))
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_one_tensor_as_both_inputs():
    """x added to itself: its gradient is the sum of both inputs'."""
    g = _gen(21)
    x, dy, dh = (_rand(g, 9, 200, dtype=F32) for _ in range(3))
    a = x.clone().requires_grad_(True)
    y, h = harp_amd.add_rms_norm(a, a)
    (got,) = torch.autograd.grad((y, h), a, (dy, dh))
    b, c = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y2, h2 = harp_amd.add_rms_norm(b, c)
    gb, gc = torch.autograd.grad((y2, h2), (b, c), (dy, dh))
    assert torch.equal(y, y2) and torch.equal(got, gb + gc)
    a = x.clone().requires_grad_(True)
    y, h = harp_amd.add_rms_norm(a, a)
    (y * dy).sum().backward(inputs=[a], retain_graph=True)
    first = a.grad.clone()
    (y * dy).sum().backward(inputs=[a])
    assert torch.equal(a.grad, 2 * first)


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)], ids=str)
@pytest.mark.parametrize("rd", [B16, F32], ids=str)
def test_gradients_of_some_inputs(need, rd):
    """Any subset of the inputs' gradients equals the one taken with all."""
    g, x, r, w = _case(6, 136, (B16, rd, F32), 4)
    dy, dh = _rand(g, 6, 136), _rand(g, 6, 136, dtype=rd)
    full = [t.clone().requires_grad_(True) for t in (x, r, w)]
    want = torch.autograd.grad(harp_amd.add_rms_norm(*full), full, (dy, dh))
    some = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, r, w), need)]
    leaves = [t for t in some if t.requires_grad]
    got = torch.autograd.grad(harp_amd.add_rms_norm(*some), leaves, (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(got, [v for v, n in zip(want, need) if n]))
    with torch.inference_mode():
        y, h = harp_amd.add_rms_norm(x, r, w)
    with torch.no_grad():
        y2, h2 = harp_amd.add_rms_norm(*some)
    assert torch.equal(y, y2) and torch.equal(h, h2) and not y2.requires_grad


def _slices(rows, *at):
    """512 rows at both ends and around each of `at`."""
    return [slice(max(0, c - 256), min(rows, c + 256)) for c in (256, *at, rows - 256)]


def test_more_rows_than_one_launch_holds():
    """A grid holds fewer than 2^32 threads: more rows run as several launches."""
    rows, cols = 2 ** 26 + 5, 8  # 4 rows in a block of 256 threads
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.empty(rows, cols, dtype=B16, device=DEV).normal_(generator=g)
    r = torch.empty(rows, cols, dtype=F32, device=DEV).normal_(generator=g)
    q = harp_amd.quantize_int8(x)
    y, h = harp_amd.add_rms_norm(x, r, None, 1e-6)
    for s in _slices(rows, 2 ** 24, 2 ** 26):
        small = harp_amd.quantize_int8(x[s])
        assert torch.equal(q.values[s], small.values) and torch.equal(q.scales[s], small.scales), s
        ys, hs = harp_amd.add_rms_norm(x[s], r[s], None, 1e-6)
        assert torch.equal(y[s], ys) and torch.equal(h[s], hs), s


def test_more_values_than_one_dequantise_launch_holds():
    rows, cols = 2 ** 25 + 3, 520  # 33 vectors of 16 values a row, 2^30 to a launch
    g = torch.Generator(DEV).manual_seed(6)
    store = torch.empty(rows, 528, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g)
    scales = torch.rand(rows, generator=g, device=DEV)
    out = harp_amd.Int8Rows(store[:, :cols], scales).dequantize(B16)
    for s in _slices(rows, 2 ** 30 // 33):
        assert torch.equal(out[s], (store[s, :cols].float() * scales[s, None]).to(B16)), s


def test_rows_whose_norm_is_not_finite():
    """eps 0 and squares that sum to 0: the normed values are infinite or NaN,
    so the scale is NaN, as every row's that holds one."""
    x = torch.zeros(4, 72, dtype=F32, device=DEV)
    x[1, 3] = 1e-30  # its square is 0 in fp32
    x[2] = 1.0
    x[3, 0] = 3e38  # its square is infinite: the normed values are 0
    y, _ = harp_amd.add_rms_norm(x, None, None, 0.0)
    rows, _ = harp_amd.add_rms_norm_int8(x, None, None, 0.0)
    assert not bool(torch.isfinite(y[:2]).all(-1).any())
    assert bool(torch.isnan(rows.scales[:2]).all()) and bool((rows.values[:2] == 0).all())
    assert bool((y[2] == 1).all()) and bool((rows.values[2] == 127).all())
    assert bool((y[3] == 0).all()) and bool((rows.dequantize(F32)[3] == 0).all())
    rows, _ = harp_amd.add_rms_norm_int8(x, None, None, 1e-6)
    assert float(rows.scales[0]) == 0.0 and bool((rows.values[0] == 0).all())


@pytest.mark.parametrize("types", TYPES[:4], ids=str)
@pytest.mark.parametrize("rows,cols", [(33, 15), (530, 33), (1000, 100), (77, 128), (2049, 8), (600, 520)])
def test_many_narrow_rows(rows, cols, types):
    """Rows that share a wave, the last ones of a block missing, in both directions and to 8 bits."""
    test_forward_backward(rows, cols, types)
    test_norm_int8(rows, cols, types[0], types[1])
    test_quantize_is_exact(rows, cols, types[0])


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tensors_of_two_devices_are_refused(which):
    for grad in (False, True):
        ts = [torch.ones(3, 64, device=DEV), torch.ones(3, 64, device=DEV), torch.ones(64, device=DEV)]
        ts[which] = ts[which].cpu()
        for t in ts:
            t.requires_grad_(grad)
        with pytest.raises(RuntimeError, match="HIP device"):
            harp_amd.add_rms_norm(*ts)


def test_forward_mode_derivatives_are_refused():
    """A tangent on any argument, or on a gradient given to the backward, raises and is not dropped."""
    import torch.autograd.forward_ad as fwAD

    from tests.test_block_abi import assert_tangents_are_refused

    assert_tangents_are_refused(DEV)
    g, x, r, w = _case(4, 72, (F32, F32, F32), 2)
    x.requires_grad_(True)
    y, h = harp_amd.add_rms_norm(x, r, w)
    with fwAD.dual_level():
        one = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
        for out in (y, h):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(out, x, one, retain_graph=True)
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool(torch.isfinite(gx).all())


def _border_rows(g, rows, scale):
    """fp32 rows with a maximum of up to `scale` and, for every border between two steps, the value nearest to it
    and that value's neighbours, either sign."""
    most = ((torch.rand(rows, 1, generator=g) + 1) * (scale / 2)).float()
    at = ((torch.arange(127, dtype=torch.float64) + 0.5) / 127 * most.double()).float()
    up, down = torch.nextafter(at, most * 2 if scale < 1e38 else most), torch.nextafter(at, torch.zeros(()))
    sign = torch.randint(0, 2, (rows, 381), generator=g) * 2.0 - 1.0
    return torch.cat([most, torch.cat([at, up, down], -1) * sign, most / 2], -1)


@pytest.mark.parametrize("scale", [2.0 ** -140, 1e-30, 2.0 ** -100, 1.0, 197.0, 1e30, 2.0 ** 121, 2.0 ** 122, 3.4e38], ids=str)
def test_quantize_beside_borders(scale):
    """fp32 values next to a border between two steps go to the nearer one, and halves to the even one.  In 64 bits
    127 x is exact and its quotient with the maximum nowhere nearer than 2^-33 to a border that it is not on."""
    x = _border_rows(_gen(7), 400, scale).to(DEV)
    if scale == 197.0:
        x[0, 0], x[0, 1:] = 196.8303680419922, 0.7749227285385132  # 0.5 + 1.3e-8 steps: 1
    q, s = harp_amd.quantize_int8(x)
    most = x.double().abs().amax(-1, keepdim=True)
    want = torch.round(127 * x.double() / most)
    assert torch.equal(q.double(), want), int((q.double() != want).sum())
    assert scale != 197.0 or bool((q[0, 1:] == 1).all())


@pytest.mark.parametrize("types", [(B16, B16, B16), (B16, None, B16), (B16, B16, None), (F32, F32, None), (B16, F32, None)],
                         ids=str)
def test_norm_int8_steps_are_exact(types):
    """The factor 1 / rms cancels from the steps: where h w is exact in fp32 (16-bit h and weight, or no weight),
    they equal those of 127 h w / max |h w| in 64 bits."""
    _, x, r, w = _case(700, 3840, types, 31)
    (q, _), h = harp_amd.add_rms_norm_int8(x, r, w, 1e-5)
    v = h.double() if w is None else h.double() * w.double()
    assert torch.equal(q.double(), torch.round(127 * v / v.abs().amax(-1, keepdim=True)))


@pytest.mark.parametrize("cols", [1, 72])
@pytest.mark.parametrize("grad", [False, True])
def test_negated_views(grad, cols):
    """The imaginary part of a conjugate is a view whose sign is turned lazily (with a stride of 2: rows of one
    value are read in place)."""
    def turned(t):
        v = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v

    g, x, r, w = _case(6, cols, (F32, F32, F32), 17)
    dy, dh = _rand(g, 6, cols, dtype=F32), _rand(g, 6, cols, dtype=F32)
    plain = [t.requires_grad_(grad) for t in (x, r, w)]
    views = [turned(t.detach()).requires_grad_(grad) for t in plain]
    want, got = harp_amd.add_rms_norm(*plain), harp_amd.add_rms_norm(*views)
    alone, alone2 = harp_amd.add_rms_norm(x, None, w), harp_amd.add_rms_norm(views[0], None, views[2])
    assert all(torch.equal(a, b) for a, b in zip((*want, *alone), (*got, *alone2)))
    if grad:
        a = torch.autograd.grad(want, plain, (dy, dh)) + torch.autograd.grad(alone[0], (x, w), dy)
        b = torch.autograd.grad(got, views, (turned(dy), turned(dh))) \
            + torch.autograd.grad(alone2[0], (views[0], views[2]), turned(dy))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x, w = x.detach(), w.detach()
    for a, b in ((harp_amd.quantize_int8(x), harp_amd.quantize_int8(turned(x))),
                 (harp_amd.add_rms_norm_int8(x, x, w)[0], harp_amd.add_rms_norm_int8(turned(x), turned(x), turned(w))[0])):
        assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)
    lin = harp_amd.Int8Linear.from_linear(torch.nn.Linear(cols, 9, device=DEV))
    with torch.no_grad():
        assert torch.equal(lin(x), lin(turned(x)))


@pytest.mark.parametrize("mode", ["grad", "no_grad", "inference"])
def test_operator_results_share_no_memory_with_x(mode):
    """The schema declares new tensors: without a residual the second is None, and the function gives x itself."""
    harp_amd.load_block_ops()
    x, w = torch.randn(4, 72, device=DEV).requires_grad_(mode == "grad"), torch.ones(72, device=DEV)
    with torch.inference_mode(mode == "inference"), torch.set_grad_enabled(mode == "grad"):
        y, h = torch.ops.harp_block.add_rms_norm(x, None, w, 1e-5)
        assert h is None
        y2, h2 = harp_amd.add_rms_norm(x, None, w, 1e-5)
        assert h2 is x and torch.equal(y, y2) and y.requires_grad == (mode == "grad")
        _, h = torch.ops.harp_block.add_rms_norm(x, x, w, 1e-5)
        assert torch.equal(h, x + x) and h.data_ptr() != x.data_ptr()


def test_more_wide_rows_than_one_launch_holds():
    """Rows with a wave each run 4 to a block, so that 2^24 fill a launch, and longer ones fill it with 2^22: what
    follows in the next launch (a row's y, h, rstd, 8-bit values and scale) is as in a call of a few rows."""
    rows, cols = 2 ** 24 + 5, 136
    g = torch.Generator(DEV).manual_seed(8)
    x = torch.empty(rows, cols, dtype=B16, device=DEV).normal_(generator=g)
    r = torch.empty(rows, cols, dtype=B16, device=DEV).normal_(generator=g)
    w = torch.rand(cols, generator=g, device=DEV) + 0.5
    q, n8 = harp_amd.quantize_int8(x), harp_amd.add_rms_norm_int8(x, r, w, 1e-6)
    x.requires_grad_(True)
    y, h = harp_amd.add_rms_norm(x, r, w, 1e-6)
    (dx,) = torch.autograd.grad((y, h), x, (r, r))
    for s in _slices(rows, 2 ** 24):
        small = harp_amd.quantize_int8(x.detach()[s])
        assert torch.equal(q.values[s], small.values) and torch.equal(q.scales[s], small.scales), s
        small, hs = harp_amd.add_rms_norm_int8(x.detach()[s], r[s], w, 1e-6)
        assert torch.equal(n8[0].values[s], small.values) and torch.equal(n8[0].scales[s], small.scales), s
        assert torch.equal(n8[1][s], hs) and torch.equal(h[s], hs), s
        xs = x.detach()[s].requires_grad_(True)
        ys, hs = harp_amd.add_rms_norm(xs, r[s], w, 1e-6)
        assert torch.equal(y[s], ys) and torch.equal(dx[s], torch.autograd.grad((ys, hs), xs, (r[s], r[s]))[0]), s
    del x, r, y, h, dx, q, n8
    rows, cols = 2 ** 22 + 3, 1040
    x = torch.empty(rows, cols, dtype=B16, device=DEV).normal_(generator=g)
    q = harp_amd.quantize_int8(x)
    for s in _slices(rows, 2 ** 22):
        small = harp_amd.quantize_int8(x[s])
        assert torch.equal(q.values[s], small.values) and torch.equal(q.scales[s], small.scales), s
