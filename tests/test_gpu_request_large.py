"""GPU tests of the operators for requests of one batch on tensors of more than
2^31 elements (4 GB and more): rows whose offsets pass 2^31 elements and 2^32
bytes, against 64 bits, and row strides beyond the 32-bit offsets of a tile."""

import math
from types import SimpleNamespace

import pytest
import torch

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {B16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()


def _normal(g, *shape, scale=1.0, dtype=B16):
    t = torch.empty(shape, dtype=dtype, device=DEV)
    return t.normal_(generator=g).mul_(scale)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(T, width, element=2):
    """Some of T rows: the first and last, those around 2^31 elements and 2^32 bytes, and others in between."""
    marks = [2 ** 31 // width, 2 ** 32 // (width * element), 2 ** 32 // width]
    picked = {0, 1, T - 2, T - 1} | {m + d for m in marks for d in (-1, 0, 1)} | set(range(T // 40, T, T // 40))
    return torch.tensor(sorted(r for r in picked if 0 <= r < T), device=DEV)


def _who(index, cuts, rows):
    request = torch.searchsorted(cuts[1:].contiguous(), rows, right=True)
    inside = (rows >= cuts[0]) & (request < index.numel())
    return torch.where(inside, index[request.clamp_max(index.numel() - 1)], -1)


def _close(got, want, size, terms, what, dtype):
    """A rounding to dtype; sums of `terms` products in 32 bits; 2^-17 of t and of its products that two parts leave."""
    tol = HALF_STEP[dtype] * want.abs() + (2.0 ** -16 + (terms + 16) * 2.0 ** -24) * size
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()))


def _requests(T, n):
    """Five requests with tokens in front of and behind them, one without an adapter."""
    cuts = torch.tensor([5, T // 7, T // 2 + 3, T // 2 + 3, T - 1000, T - 9], dtype=torch.int64, device=DEV)
    return torch.tensor([1, 0, 1, -1, n - 1], device=DEV), cuts


@pytest.mark.parametrize("N,dtype,each", [(2312, B16, False), (2311, B16, False), (2312, F32, False), (2312, B16, True)])
def test_a_projection_s_result(N, dtype, each):
    """tokens x features past 2^31; `each`: a request of four tokens, 2^18 of them."""
    g = _gen(N)
    T, K, r, n = 2 ** 20 + 4, 72, 16, 3
    assert T * N > 2 ** 31
    x, base = _normal(g, T, K), _normal(g, T, N, dtype=dtype)
    low = harp_amd.Adapters(_normal(g, n, r, K, scale=K ** -0.5), _normal(g, n, N, r, scale=0.5 * r ** -0.5))
    if each:
        index, cuts = torch.arange(T // 4, device=DEV) % (n + 1) - 1, torch.arange(T // 4 + 1, device=DEV) * 4
        requests = harp_amd.AdapterRequests(index)
    else:
        index, cuts = _requests(T, n)
        requests = harp_amd.AdapterRequests(index, cuts)
    out = harp_amd.add_adapters(base, x, low, requests)
    rows = _rows(T, N, base.element_size())
    who = _who(index, cuts, rows)
    for which in range(-1, n):
        mine = rows[who == which]
        if not mine.numel():
            continue
        if which < 0:
            assert torch.equal(out[mine], base[mine])
            continue
        xd, a, b = x[mine].double(), low.a[which].double(), low.b[which].double()
        want = base[mine].double() + xd @ a.t() @ b.t()
        _close(out[mine], want, base[mine].double().abs() + xd.abs() @ a.abs().t() @ b.abs().t(), K + r, which, dtype)
    # the rows that no request has, all of them
    assert torch.equal(out[:int(cuts[0])], base[:int(cuts[0])]) and torch.equal(out[int(cuts[-1]):], base[int(cuts[-1]):])


@pytest.mark.parametrize("K", [2312, 2311])
def test_a_wide_input_and_its_gradients(K):
    """tokens x columns past 2^31, forward and backward.  Only some rows of x and dy are not zero, so that the
    weights' gradients are short sums and a row read from another place would be missed in them."""
    g = _gen(K)
    T, N, r, n = 2 ** 20 + 4, 40, 16, 3
    rows = _rows(T, K)
    x = torch.zeros(T, K, dtype=B16, device=DEV)
    x[rows] = _normal(g, rows.numel(), K)
    dy = torch.zeros(T, N, dtype=B16, device=DEV)
    dy[rows] = _normal(g, rows.numel(), N)
    base = _normal(g, T, N)
    low = harp_amd.Adapters(_normal(g, n, r, K, scale=K ** -0.5).requires_grad_(),
                            _normal(g, n, N, r, scale=0.5 * r ** -0.5).requires_grad_())
    index, cuts = _requests(T, n)
    out = harp_amd.add_adapters(base, x.requires_grad_(), low, harp_amd.AdapterRequests(index, cuts))
    dx, da, db = torch.autograd.grad(out, (x, low.a, low.b), dy)
    who = _who(index, cuts, rows)
    assert torch.equal(out[rows[who < 0]], base[rows[who < 0]]) and not bool(dx[rows[who < 0]].any())
    for which in range(n):
        mine = rows[who == which]
        assert mine.numel()
        xd, d, a, b = x[mine].detach().double(), dy[mine].double(), low.a[which].detach().double(), low.b[which].detach().double()
        xs, ds, sa, sb = xd.abs(), d.abs(), a.abs(), b.abs()
        t, u = xd @ a.t(), d @ b
        ts, us = xs @ sa.t(), ds @ sb
        _close(out[mine].detach(), base[mine].double() + t @ b.t(), base[mine].double().abs() + ts @ sb.t(), K + r, "out", B16)
        _close(dx[mine], u @ a, us @ sa, N + r, "dx", B16)
        _close(da[which], u.t() @ xd, us.t() @ xs, N + mine.numel(), "da", B16)
        _close(db[which], d.t() @ t, ds.t() @ ts, K + mine.numel(), "db", B16)
    others = torch.ones(T, dtype=torch.bool, device=DEV)
    others[rows] = False
    assert float(dx.abs().amax(1)[others].max()) == 0.0


def test_row_strides_beyond_a_tile_s_offsets():
    """x, base and dy as columns of tensors with 2^24 + 8 elements a row."""
    g = _gen(3)
    T, K, N, r, n, wide = 140, 72, 136, 16, 2, 2 ** 24 + 8
    store = torch.empty(T, wide, dtype=B16, device=DEV)
    x, base, dy = store[:, 8:8 + K], store[:, 1024:1024 + N], store[:, wide - N:]
    for t in (x, base, dy):
        t.copy_(_normal(g, *t.shape))
    low = harp_amd.Adapters(_normal(g, n, r, K, scale=K ** -0.5).requires_grad_(),
                            _normal(g, n, N, r, scale=0.5 * r ** -0.5).requires_grad_())
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
    results = []
    for form in (lambda t: t, lambda t: t.contiguous()):
        xs = form(x).detach().requires_grad_()
        out = harp_amd.add_adapters(form(base), xs, low, requests)
        results.append((out, *torch.autograd.grad(out, (xs, low.a, low.b), form(dy))))
    # (x is read by another kernel where the stride is large, in another order: 32-bit sums of K and N products)
    for a, b in zip(*results):
        d = (a.detach().double() - b.detach().double()).abs()
        assert float(d.max()) <= 2.0 ** -7 * float(b.detach().double().abs().max())
        assert float((d > 0).float().mean()) <= 2.0 ** -6


@pytest.mark.parametrize("dtype,half,H,D", [(B16, False, 20, 128), (B16, True, 34, 64), (F32, False, 9, 256)])
def test_rotation_of_many_rows(dtype, half, H, D):
    """q past 2^31 elements beside a k of one head, token-major, forward and backward."""
    g = _gen(D)
    S = 2 ** 20 + 2
    assert S * H * D > 2 ** 31
    rope = harp_amd.AxialRope((D // 4, D // 4, D // 2), 256.0, "half" if half else "interleaved")
    q = _normal(g, 1, S, H, D, dtype=dtype).transpose(1, 2).requires_grad_()
    k = _normal(g, 1, S, 1, D, dtype=dtype).transpose(1, 2)
    w = (1 + 0.1 * torch.randn(D, device=DEV, generator=g)).to(dtype)
    pos = torch.randint(0, 4000, (S, 3), device=DEV, generator=g, dtype=torch.int32)
    y, yk = harp_amd.qk_norm_axial_rope(q, k, pos, rope, w, None, (1e-5, None))
    dy = _normal(g, 1, S, H, D, dtype=dtype).transpose(1, 2)
    (dx,) = torch.autograd.grad(y, q, dy)
    rows = _rows(S, H * D, q.element_size())
    ang = torch.cat([pos[rows, a, None].double() * 256.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
                     for a, d in enumerate(rope.axes_dims)], -1)
    c, s = torch.cos(ang), torch.sin(ang)

    def turn(v, c, s):
        a, b = v.chunk(2, -1) if half else (v[..., 0::2], v[..., 1::2])
        v = torch.stack((a * c - b * s, a * s + b * c), -1)
        return v.transpose(-1, -2).flatten(-2) if half else v.flatten(-2)

    def close(got, want, slack):  # a rounding, and 2^-19 of the terms (32 steps of 32 bits)
        tol = HALF_STEP[dtype] * want.abs() + 2.0 ** -19 * slack
        assert not bool(((got.double() - want).abs() > tol).any())

    x, d = (t[0][:, rows].detach().double() for t in (q, dy))
    rho = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    n = x * rho
    big = (n * w.double()).abs().amax(-1, keepdim=True)
    close(y.detach()[0][:, rows], turn(n * w.double(), c, s), 2 * big)
    gr = turn(d, c, -s) * w.double()
    want = rho * (gr - n * (gr * n).mean(-1, keepdim=True))
    close(dx[0][:, rows], want, 4 * rho * gr.abs().amax(-1, keepdim=True) * (1 + n.abs().amax(-1, keepdim=True) ** 2))
    kd = k[0][:, rows].double()
    close(yk[0][:, rows], turn(kd, c, s), 2 * kd.abs().amax(-1, keepdim=True))
    assert math.isfinite(float(dx.float().abs().max() if dtype == F32 else dx.abs().max()))


def test_projections_of_more_tokens_than_adapters_take():
    """2^25 tokens and more: without requests the parts run; with them the adapters' limit is named."""
    g = _gen(5)
    S, dim = 2 ** 25 + 128, 64
    attn = SimpleNamespace(heads=1)
    for name in ("to_q", "to_k", "to_v"):
        setattr(attn, name, torch.nn.Linear(dim, 128, bias=False, dtype=B16, device=DEV).requires_grad_(False))
    attn.norm_q = attn.norm_k = SimpleNamespace(weight=torch.ones(128, dtype=B16, device=DEV), eps=1e-5)
    low = {name: harp_amd.Adapters(_normal(g, 2, 8, dim), _normal(g, 2, 128, 8)) for name in ("to_q", "to_k", "to_v")}
    attn = harp_amd.adapt_attention(attn, **low)
    x = _normal(g, 1, S, dim)
    rope = harp_amd.AxialRope((32, 48, 48), 256.0)
    pos = torch.randint(0, 4000, (S, 3), device=DEV, generator=g, dtype=torch.int32)
    with torch.no_grad():
        q, _, v = harp_amd.project_qkv(attn, x, harp_amd.AxialPositions(pos, rope))
        for at in (slice(0, 300), slice(S - 300, S)):
            few = harp_amd.project_qkv(attn, x[:, at].contiguous(), harp_amd.AxialPositions(pos[at].contiguous(), rope))
            # (parts round three times, the one launch once: 0.5 * 2^-8 of the norm each at most)
            for a, b in ((q, few[0]), (v, few[2])):
                assert float((a[:, :, at].double() - b.double()).norm() / b.double().norm()) <= 6e-3
        with pytest.raises(RuntimeError, match="2\\^25"):
            harp_amd.project_qkv(attn, x, harp_amd.AxialPositions(pos, rope),
                                 requests=harp_amd.AdapterRequests(torch.zeros(1, dtype=torch.int32, device=DEV)))
