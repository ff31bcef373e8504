"""GPU tests of the QK RMSNorm with rotary positions of several axes, forward
and backward, and of the rotary table, against the formulas in 64 bits."""

import decimal
import math

import pytest
import torch

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {B16: 2.0 ** -8, F32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, scale=1.0, dtype=B16):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _heads(g, B, S, H, D, dtype):
    """[B, H, S, D] over token-major storage, as a projection gives it."""
    return _rand(g, B, S, H, D, dtype=dtype).transpose(1, 2)


def _angles(positions, rope):
    """[B or 1, 1, S, D / 2] in 64 bits."""
    parts = []
    for a, (d, theta) in enumerate(zip(rope.axes_dims, rope.theta)):
        j = torch.arange(d // 2, dtype=torch.float64, device=positions.device)
        parts.append(positions[..., a, None].double() * theta ** (-2 * j / d))
    ang = torch.cat(parts, -1)
    return ang[:, None] if ang.dim() == 3 else ang[None, None]


def _pairs(x, half):
    if half:
        return x.unflatten(-1, (2, -1)).transpose(-1, -2)
    return x.unflatten(-1, (-1, 2))


def _unpairs(x, half):
    return x.transpose(-1, -2).flatten(-2) if half else x.flatten(-2)


def _turn(x, ang, half):
    p = _pairs(x, half)
    c, s = torch.cos(ang), torch.sin(ang)
    return _unpairs(torch.stack((p[..., 0] * c - p[..., 1] * s, p[..., 0] * s + p[..., 1] * c), -1), half)


def _pair_size(x, half):
    """|x0| + |x1| of each element's pair: what its rotation's terms are made of."""
    return _unpairs(_pairs(x.abs(), half).sum(-1, keepdim=True).expand(*x.shape[:-1], x.shape[-1] // 2, 2), half)


def _close(got, want, dtype, slack, what):
    """One rounding to dtype, and 32-bit arithmetic: 2^-19 (32 steps of 2^-24) of the terms, ``slack``."""
    tol = HALF_STEP[dtype] * want.abs() + 2.0 ** -19 * slack + 1e-30
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def _rms(x, eps):
    return 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)


def _check_forward(y, x, w, eps, ang, half):
    x = x.detach().double()
    if eps is not None:
        x = x * _rms(x, eps) * (1.0 if w is None else w.detach().double())
    _close(y.detach(), _turn(x, ang, half), y.dtype, _pair_size(x, half), "y")


def _check_backward(dx, dw, dy, x, w, eps, ang, half):
    d = _turn(dy.double(), -ang, half)
    size = _pair_size(dy.double(), half)
    if eps is None:
        _close(dx, d, dx.dtype, size, "dx")
        return
    x = x.detach().double()
    r = _rms(x, eps)
    n = x * r
    wd = 1.0 if w is None else w.detach().double()
    g = d * wd
    mean = (g * n).mean(-1, keepdim=True)
    small = (size * (wd if w is None else wd.abs()) * n.abs()).mean(-1, keepdim=True)
    _close(dx, r * (g - n * mean), dx.dtype, r * (size * (wd if w is None else wd.abs()) + n.abs() * small), "dx")
    if dw is not None:
        rows = d.numel() // d.shape[-1]
        want = (d * n).sum((0, 1, 2))
        # a sum of `rows` terms in 32 bits is off by at most rows * 2^-24 of their sizes, and each term by 32 steps
        tol = HALF_STEP[dw.dtype] * want.abs() + (rows + 32) * 2.0 ** -24 * (size * n.abs()).sum((0, 1, 2))
        assert bool(((dw.double() - want).abs() <= tol).all())


def _axes(D):
    t = D // 8 * 2
    h = (D - t) // 4 * 2
    return (t, h, D - t - h)


def _grid(S, g, B=None, dtype=torch.int32):
    shape = (S, 3) if B is None else (B, S, 3)
    p = torch.randint(-50, 2000, shape, generator=g)
    return (p.float() * 0.37 if dtype == F32 else p.to(dtype)).to(DEV)


CASES = [
    # B, S, Hq, Hk, D, dtype, half, positions, each, norm
    (1, 1, 1, 1, 8, B16, False, torch.int32, False, True),
    (2, 1, 30, 30, 128, B16, False, torch.int32, True, True),
    (1, 7, 3, 1, 16, B16, True, torch.int64, False, True),
    (2, 33, 5, 2, 64, B16, False, F32, True, True),
    (3, 19, 4, 4, 72, F32, True, torch.int32, False, True),
    (1, 300, 14, 2, 128, B16, True, torch.int64, True, True),
    (2, 65, 3, 3, 136, B16, False, torch.int32, True, True),
    (1, 41, 2, 7, 256, F32, False, F32, False, True),
    (1, 50, 6, 3, 40, F32, False, torch.int64, True, True),
    (1, 21, 2, 2, 128, B16, False, torch.int32, False, False),
    (2, 13, 3, 1, 248, F32, True, F32, True, False),
    (1, 2100, 30, 30, 128, B16, False, torch.int32, False, True),   # four heads to a group
    (1, 700, 30, 30, 64, B16, True, torch.int32, False, True),      # two heads to a group
    (1, 1500, 29, 3, 256, B16, False, torch.int32, False, True),    # an odd number of heads
]


@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,half,pos,each,norm", CASES)
def test_forward_and_backward(B, S, Hq, Hk, D, dtype, half, pos, each, norm):
    g = _gen(S * D + Hq)
    rope = harp_amd.AxialRope(_axes(D), 256.0, "half" if half else "interleaved")
    positions = _grid(S, g, B if each else None, pos)
    q, k = (_heads(g, B, S, H, D, dtype).requires_grad_() for H in (Hq, Hk))
    wq = (1 + _rand(g, D, scale=0.1, dtype=F32)).to(B16).requires_grad_() if norm else None
    wk = (1 + _rand(g, D, scale=0.1, dtype=F32)).requires_grad_() if norm else None
    eps = 1e-5 if norm else None
    yq, yk = harp_amd.qk_norm_axial_rope(q, k, positions, rope, wq, wk, eps)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.stride() == q.stride() and yk.stride() == k.stride()
    ang = _angles(positions, rope)
    _check_forward(yq, q, wq, eps, ang, half)
    _check_forward(yk, k, wk, eps, ang, half)
    dq, dk = (_heads(g, B, S, H, D, dtype) for H in (Hq, Hk))
    got = torch.autograd.grad((yq, yk), (q, k) + ((wq, wk) if norm else ()), (dq, dk))
    _check_backward(got[0], got[2] if norm else None, dq, q, wq, eps, ang, half)
    _check_backward(got[1], got[3] if norm else None, dk, k, wk, eps, ang, half)


@pytest.mark.parametrize("axes,theta", [((128,), 1e4), ((64, 64), (256.0, 1e6)), ((2, 2, 2, 2), 10.0),
                                        ((16, 40, 40, 32), (1e4, 256.0, 10.0, 2.0))])
def test_axes(axes, theta):
    g = _gen(len(axes))
    rope = harp_amd.AxialRope(axes, theta)
    D, S = sum(axes), 57
    positions = torch.randint(0, 3000, (S, len(axes)), generator=g).to(DEV)
    q = _heads(g, 2, S, 3, D, F32)
    y, none = harp_amd.qk_norm_axial_rope(q, None, positions, rope)
    assert none is None
    _check_forward(y, q, None, None, _angles(positions, rope), False)
    table = rope.table(positions)
    ang = _angles(positions, rope)[0, 0]
    assert table.dtype == torch.complex64 and table.shape == (S, D // 2)
    assert float((table.to(torch.complex128) - torch.polar(torch.ones_like(ang), ang)).abs().max()) <= 2.0 ** -21


def test_table_of_a_batch_and_strided_positions():
    g = _gen(3)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    store = torch.randint(0, 900, (3, 40, 6), generator=g).to(DEV)
    positions = store.transpose(0, 1).transpose(0, 1)[..., ::2]
    a = rope.table(positions)
    assert a.shape == (3, 40, 64)
    assert torch.equal(a, rope.table(positions.contiguous())) and torch.equal(a[1], rope.table(positions[1].int()))
    assert harp_amd.AxialPositions(positions, rope).table().equal(a)
    empty = rope.table(torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    assert empty.shape == (0, 64)


def test_far_positions_keep_their_precision():
    """Positions near 2^31, fractions of 2^20: angles of 32 bits would be off by whole turns."""
    rope = harp_amd.AxialRope((8, 8), 100.0)
    p = torch.tensor([[2 ** 31 - 1, -2 ** 31], [2 ** 30 + 7, 2 ** 24 + 1], [-5, 123456789]], device=DEV)
    ang = torch.cat([p[:, a, None].cpu().double() * 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
                     for a in (0, 1)], -1)
    want = torch.polar(torch.ones_like(ang), ang)
    got = rope.table(p.int().to(DEV)).to(torch.complex128).cpu()
    # the angle: 64-bit products of up to 2^28.4 turns, off by 2^-24 of a turn
    assert float((got - want).abs().max()) <= 2 * math.pi * 2.0 ** -23 + 2.0 ** -21
    fine = torch.tensor([[1048575.75, 0.25]], device=DEV)
    ang = torch.cat([fine[:, a, None].cpu().double() * 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
                     for a in (0, 1)], -1)
    got = rope.table(fine).to(torch.complex128).cpu()
    assert float((got - torch.polar(torch.ones_like(ang), ang)).abs().max()) <= 2.0 ** -21


@pytest.mark.parametrize("axes,theta", [((100, 20, 8), 1e6), ((32, 48, 48), 256.0), ((2, 2, 252), 1e6), ((16, 56, 56), 1e4),
                                        ((128,), 1e4), ((64, 64), (1.0, 1e6))])
def test_far_positions_along_the_axes_behind_others(axes, theta):
    """Positions near 2^31 along every axis: the angle is off by 2^-22 of a turn at most, whatever axes are in
    front.  The angles in whole numbers and 60 digits; 2^-21 is the 32-bit sine's and cosine's own."""
    rope = harp_amd.AxialRope(axes, theta)
    values = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 12345, 2 ** 30 + 7, -1999999999]
    p = torch.tensor(values)[:, None].expand(-1, len(axes)).to(torch.int32)
    with decimal.localcontext() as c:
        c.prec = 60
        two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        want = []
        for v in values:
            row = []
            for d, th in zip(axes, rope.theta):
                for j in range(d // 2):
                    turns = v * (decimal.Decimal(th).ln() * (-2 * j) / d).exp() / two_pi
                    row.append(float((turns - turns.to_integral_value()) * two_pi))
            want.append(row)
    ang = torch.tensor(want, dtype=torch.float64)
    got = rope.table(p.to(DEV)).to(torch.complex128).cpu()
    assert float((got - torch.polar(torch.ones_like(ang), ang)).abs().max()) <= 2 * math.pi * 2.0 ** -22 + 2.0 ** -21


def test_quarter_turns_are_exact():
    """Every multiple of an eighth of a turn in both directions: the branches of the reduction."""
    rope = harp_amd.AxialRope((2, 2, 2, 2), 1.0)
    turns = torch.arange(-64, 65, dtype=torch.float64) / 16
    p = (turns * 2 * math.pi).float()[:, None].expand(-1, 4).contiguous().to(DEV)
    ang = p[:, :4].double().cpu()
    got = rope.table(p).to(torch.complex128).cpu()
    assert float((got - torch.polar(torch.ones_like(ang), ang)).abs().max()) <= 2.0 ** -21


def _view(x, kind):
    """The same values in another layout."""
    if kind == "expanded":
        return x[:1].expand(x.size(0), -1, -1, -1)
    if kind == "head_major":
        return x.contiguous()
    if kind == "padded":  # rows of a wider tensor: strides that are multiples of 8
        store = torch.zeros(*x.shape[:3], x.size(3) + 24, dtype=x.dtype, device=DEV)
        store[..., 8:8 + x.size(3)] = x
        return store[..., 8:8 + x.size(3)]
    if kind == "odd":  # neither 16-byte aligned nor strides of 8
        store = torch.zeros(*x.shape[:3], x.size(3) + 3, dtype=x.dtype, device=DEV)
        store[..., 1:1 + x.size(3)] = x
        return store[..., 1:1 + x.size(3)]
    if kind == "column":  # features are not neighbours
        return x.transpose(2, 3).contiguous().transpose(2, 3)
    return torch._neg_view(-x)


@pytest.mark.parametrize("kind", ["expanded", "head_major", "padded", "odd", "column", "negated"])
def test_layouts(kind):
    g = _gen(11)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    positions = _grid(37, g, 2)
    q = _heads(g, 2, 37, 3, 128, B16)
    if kind == "expanded":
        q = q[:1].repeat(2, 1, 1, 1)
    w = (1 + _rand(g, 128, scale=0.1, dtype=F32)).to(B16)
    d = _heads(g, 2, 37, 3, 128, B16)
    want, got = [], []
    for xs, ds, out in ((q, d, want), (_view(q, kind), _view(d, kind) if kind != "expanded" else d, got)):
        xs = xs.detach().requires_grad_() if not xs.is_neg() else xs
        y, _ = harp_amd.qk_norm_axial_rope(xs, None, positions, rope, w, None, 1e-5)
        out.append(y.detach())
        if xs.requires_grad:
            out.append(torch.autograd.grad(y, xs, ds)[0])
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("dtype", [B16, F32])
def test_contiguous_tensors_from_any_address_on(dtype, offset):
    """q, k and their results' gradients as parts of a packed buffer: contiguous, but not 16-byte aligned."""
    g = _gen(17 + offset)
    rope = harp_amd.AxialRope((8, 4, 4), 256.0)
    B, S, H, D = 2, 9, 3, 16
    size = B * H * S * D

    def packed(t):
        store = torch.zeros(size + 8, dtype=dtype, device=DEV)
        store[offset:offset + size] = t.flatten()
        return store[offset:offset + size].view(B, H, S, D)

    q, k, dq, dk = (_rand(g, B, H, S, D, dtype=dtype) for _ in range(4))
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(DEV)
    pos = _grid(S, g).to(DEV)
    results = []
    for form in (lambda t: t.clone(), packed):
        x = [form(t).requires_grad_() for t in (q, k)]
        d = [form(t) for t in (dq, dk)]
        assert all(t.is_contiguous() for t in (*x, *d))
        for eps in (1e-5, None):
            out = harp_amd.qk_norm_axial_rope(*x, pos, rope, *((w, w) if eps else ()), eps=eps)
            results.append((*out, *torch.autograd.grad(out, x, d)))
    for a, b in zip(results[0] + results[1], results[2] + results[3]):
        assert torch.equal(a, b)


def test_results_have_the_layout_of_q_and_k():
    """Token-major, head-major, parts of one packed projection, rows that are no multiple of 16 bytes apart: the
    order of q's and k's dimensions, without holes."""
    g = _gen(23)
    B, S, H, D = 2, 6, 3, 16
    rope = harp_amd.AxialRope((4, 4, 8), 256.0)
    pos = _grid(S, g).to(DEV)
    token, head = (S * H * D, D, H * D, 1), (H * S * D, S * D, D, 1)
    packed = _rand(g, B, S, 3, H, D).requires_grad_()
    odd = _rand(g, B, S, H, D + 3)[..., 1:1 + D].transpose(1, 2)
    forms = [(_heads(g, B, S, H, D, B16), token), (_rand(g, B, H, S, D), head), (odd, token),
             *((packed[:, :, i].transpose(1, 2), token) for i in range(3)),
             (_rand(g, B, S, 1, D).expand(-1, -1, H, -1).transpose(1, 2), None),
             (_rand(g, B, H, D, S).transpose(2, 3), head)]
    for x, strides in forms:
        y, yk = harp_amd.qk_norm_axial_rope(x, x, pos, rope, eps=1e-5)
        want, _ = harp_amd.qk_norm_axial_rope(x.detach().clone(memory_format=torch.contiguous_format), None, pos, rope, eps=1e-5)
        assert torch.equal(y, want) and torch.equal(yk, want) and y.stride(3) == 1
        assert strides is None or (y.stride() == strides and yk.stride() == strides)
    q, k = (packed[:, :, i].transpose(1, 2) for i in (0, 1))
    out = harp_amd.qk_norm_axial_rope(q, k, pos, rope, eps=1e-5)
    (grad,) = torch.autograd.grad(out, packed, [torch.ones_like(t) for t in out])
    leaves = [t.detach().clone().requires_grad_() for t in (q, k)]
    same = harp_amd.qk_norm_axial_rope(*leaves, pos, rope, eps=1e-5)
    for i, d in enumerate(torch.autograd.grad(same, leaves, [torch.ones_like(t) for t in same])):
        assert torch.equal(grad[:, :, i].transpose(1, 2), d)
    assert not bool(grad[:, :, 2].any())


def test_rows_that_are_empty_zero_or_not_finite():
    g = _gen(5)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    for shape in ((0, 3, 5, 128), (2, 0, 5, 128), (2, 3, 0, 128)):
        x = torch.zeros(shape, dtype=B16, device=DEV, requires_grad=True)
        w = torch.ones(128, dtype=B16, device=DEV, requires_grad=True)
        p = torch.zeros(shape[2], 3, dtype=torch.int32, device=DEV)
        y, _ = harp_amd.qk_norm_axial_rope(x, None, p, rope, w, None, 1e-5)
        assert y.shape == x.shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert gx.shape == x.shape and bool((gw == 0).all())
    x = _heads(g, 1, 6, 2, 128, B16)
    x[0, 0, 2] = 0
    x[0, 1, 3, 5] = float("inf")
    x[0, 0, 4, 7] = float("nan")
    p = _grid(6, g)
    y, _ = harp_amd.qk_norm_axial_rope(x, None, p, rope, None, None, 1e-6)
    assert bool((y[0, 0, 2] == 0).all())
    bad = torch.zeros(1, 2, 6, dtype=torch.bool, device=DEV)
    bad[0, 1, 3] = bad[0, 0, 4] = True
    assert bool((y.isnan().any(-1) == bad).all()) and bool(y[~bad].isfinite().all())
    far = torch.tensor([[float("inf"), 0.0, 0.0]], device=DEV)
    y, _ = harp_amd.qk_norm_axial_rope(x[:, :, :1], None, far, rope)
    assert bool(y[..., :32].isnan().all()) and torch.equal(y[..., 32:], x[:, :, :1, 32:])


@pytest.mark.parametrize("eps", [(1e-5, None), (None, 1e-6)])
def test_a_norm_of_one_of_the_two(eps):
    g = _gen(17)
    rope = harp_amd.AxialRope((16, 24, 24), 256.0)
    p = _grid(90, g)
    q, k = (_heads(g, 2, 90, H, 64, B16).requires_grad_() for H in (4, 2))
    w = (1 + _rand(g, 64, scale=0.1, dtype=F32)).requires_grad_()
    ws = tuple(w if e is not None else None for e in eps)
    out = harp_amd.qk_norm_axial_rope(q, k, p, rope, *ws, eps)
    ang = _angles(p, rope)
    d = [_heads(g, 2, 90, H, 64, B16) for H in (4, 2)]
    gq, gk, gw = torch.autograd.grad(out, (q, k, w), d)
    for y, x, dx, dy, wi, e in zip(out, (q, k), (gq, gk), d, ws, eps):
        _check_forward(y, x, wi, e, ang, False)
        _check_backward(dx, gw if wi is not None else None, dy, x, wi, e, ang, False)


def test_one_result_without_a_gradient():
    g = _gen(23)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    p = _grid(40, g)
    q, k = (_heads(g, 1, 40, H, 128, B16).requires_grad_() for H in (3, 2))
    w = torch.ones(128, dtype=B16, device=DEV, requires_grad=True)
    yq, yk = harp_amd.qk_norm_axial_rope(q, k, p, rope, w, None, 1e-5)
    d = _heads(g, 1, 40, 2, 128, B16)
    gq, gk, gw = torch.autograd.grad(yk, (q, k, w), d, allow_unused=True)
    assert gq is None and gw is None
    _check_backward(gk, None, d, k, None, 1e-5, _angles(p, rope), False)


def test_gradient_against_differences():
    """The fp32 gradient against central differences of the fp32 forward, whose
    own error is 2^-24 of a result of a few units over a step of 2^-6, and the
    third derivative's step^2 / 6: 1e-3 of the directional derivative's terms."""
    g = _gen(29)
    rope = harp_amd.AxialRope((16, 24, 24), 256.0)
    p = _grid(9, g)
    q = _heads(g, 1, 9, 2, 64, F32).requires_grad_()
    w = (1 + _rand(g, 64, scale=0.1, dtype=F32)).requires_grad_()
    d = _heads(g, 1, 9, 2, 64, F32)

    def loss(x, v):
        return float((harp_amd.qk_norm_axial_rope(x, None, p, rope, v, None, 1e-5)[0].double() * d.double()).sum())

    y, _ = harp_amd.qk_norm_axial_rope(q, None, p, rope, w, None, 1e-5)
    gx, gw = torch.autograd.grad(y, (q, w), d)
    step = 2.0 ** -6
    with torch.no_grad():
        for seed in range(3):
            vx, vw = _heads(_gen(seed), 1, 9, 2, 64, F32), _rand(_gen(seed + 9), 64, dtype=F32)
            for along, got in ((vx, (gx.double() * vx.double()).sum()), (vw, (gw.double() * vw.double()).sum())):
                if along is vx:
                    diff = (loss(q + step * vx, w) - loss(q - step * vx, w)) / (2 * step)
                else:
                    diff = (loss(q, w + step * vw) - loss(q, w - step * vw)) / (2 * step)
                terms = float((d.abs().double() * 2).sum()) / 8
                assert abs(diff - float(got)) <= 1e-3 * terms, (diff, float(got))


def test_refusals():
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    q = torch.zeros(1, 2, 4, 128, dtype=B16, device=DEV)
    p = torch.zeros(4, 3, dtype=torch.int32, device=DEV)
    f = harp_amd.qk_norm_axial_rope
    for args, msg in [
        ((q.half(), None, p, rope), "bfloat16 or float32"),
        ((q[0], None, p, rope), r"\[B, heads, S, D\]"),
        ((q[..., :64], None, p, rope), "the axes 128"),
        ((q, q.float(), p, rope), "as q"),
        ((q, q[:, :, :3], p, rope), "k must be"),
        ((q, None, p[:3], rope), "positions must be"),
        ((q, None, p[:, :2], rope), "positions must be"),
        ((q, None, p.to(torch.int16), rope), "int32, int64 or float32"),
        ((q, None, p.cpu(), rope), "positions must be on"),
        ((q, None, p, rope, torch.ones(128, device=DEV)), "eps is missing"),
        ((q, None, p, rope, torch.ones(64, device=DEV), None, 1e-5), "vector of 128"),
        ((q, None, p, rope, torch.ones(128, dtype=torch.half, device=DEV), None, 1e-5), "bfloat16 or float32"),
        ((q, None, p, rope, None, torch.ones(128, device=DEV), 1e-5), "without k"),
        ((torch.zeros(1, 2, 4, 12, dtype=B16, device=DEV), None, p, harp_amd.AxialRope((4, 4, 4), 10.0)), "multiple of 8"),
        ((torch.zeros(1, 2, 4, 264, dtype=B16, device=DEV), None, p, harp_amd.AxialRope((88, 88, 88), 10.0)), "at most 256"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            f(*args)
    with pytest.raises(RuntimeError, match="no gradient here"):
        f(q, None, p.float().requires_grad_(), rope)
    with pytest.raises(RuntimeError, match="no gradient here"):
        rope.table(p.float().requires_grad_())
    x = q.clone().requires_grad_()
    y, _ = f(x, None, p, rope, None, None, 1e-5)
    g, = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.float().sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(torch.autograd.forward_ad.make_dual(q, q), None, p, rope)
