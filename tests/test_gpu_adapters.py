"""GPU tests of low-rank adapters beside a projection, forward and backward,
against the formulas in 64 bits."""

import pytest
import torch

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {B16: 2.0 ** -8, F32: 2.0 ** -24}
STEP32 = 2.0 ** -23  # one addition of a 32-bit sum on the matrix cores


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, scale=1.0, dtype=B16):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _low(g, n, r, K, N):
    scales = (torch.rand(n, generator=g) + 0.5).to(DEV)
    return harp_amd.Adapters(_rand(g, n, r, K, scale=K ** -0.5), _rand(g, n, N, r, scale=r ** -0.5), scales)


def _segments(requests, T):
    index = requests.index.tolist()
    if requests.offsets is None:
        L = T // len(index)
        return [(i * L, (i + 1) * L, a) for i, a in enumerate(index)]
    o = [min(max(v, 0), T) for v in requests.offsets.tolist()]
    return [(o[i], o[i + 1], a) for i, a in enumerate(index)]


def _low_sum(x, low, n, requests):
    """t = s x A^T of each token and what its 32-bit sum may be off by."""
    a, _, s = low
    t = torch.zeros(x.size(0), a.size(1), dtype=torch.float64, device=DEV)
    off = torch.zeros_like(t)
    for b, e, i in _segments(requests, x.size(0)):
        if 0 <= i < n and e > b:
            sc = 1.0 if s is None else float(s[i])
            xd, ad = x[b:e].double(), a[i].double()
            t[b:e] = sc * (xd @ ad.t())
            off[b:e] = sc * (a.size(2) + 8) * STEP32 * (xd.abs() @ ad.abs().t())
    return t, off


def _per_token(v, off, mats, n, requests, parts):
    """v M_i of each token's adapter, M_i [r, C], and its error: v's own, what `parts` bf16 leave of v, the sum's."""
    C = mats.size(2)
    y = torch.zeros(v.size(0), C, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    for b, e, i in _segments(requests, v.size(0)):
        if 0 <= i < n and e > b:
            m = mats[i].double()
            y[b:e] = v[b:e] @ m
            left = off[b:e] + 2.0 ** (-8 * parts - parts + 1) * v[b:e].abs()
            err[b:e] = left @ m.abs() + (parts * v.size(1) + 8) * STEP32 * (v[b:e].abs() @ m.abs())
    return y, err


def _within(got, want, err, what):
    tol = HALF_STEP[got.dtype] * (want.abs() + err) + err + 1e-30
    ratio = ((got.double() - want).abs() / tol).max() if got.numel() else torch.zeros(())
    assert float(ratio) <= 1, (what, float(ratio))


def _check(base, x, low, requests, out, dy=None, grads=None):
    n, r = low.a.size(0), low.a.size(1)
    T, N = x.numel() // x.size(-1), base.size(-1)
    x2 = x.detach().reshape(T, -1)
    a, b = low.a.detach(), low.b.detach()
    t, off = _low_sum(x2, (a, b, low.scales), n, requests)
    y, err = _per_token(t, off, b.transpose(1, 2), n, requests, 3 if base.dtype == F32 else 2)
    want = base.detach().reshape(T, N).double() + y
    _within(out.detach().reshape(T, N), want, err + 2.0 ** -24 * want.abs(), "out")
    if dy is None:
        return
    gx, ga, gb = grads
    d2 = dy.reshape(T, N)
    u, uoff = _low_sum(d2, (b.transpose(1, 2), None, low.scales), n, requests)
    gx_want, gx_err = _per_token(u, uoff, a, n, requests, 2)
    _within(gx.reshape(T, -1), gx_want, gx_err, "dx")
    for got, left, loff, right, flip in ((ga, u, uoff, x2, False), (gb, t, off, d2, True)):
        for i in range(n):
            rows = [m for s, e, j in _segments(requests, T) if j == i for m in range(s, e)]
            v, vo, w = left[rows], loff[rows], right[rows].double()
            g = v.t() @ w
            e = vo.t() @ w.abs() + (len(rows) + 8) * STEP32 * (v.abs().t() @ w.abs())
            _within(got[i], g.t() if flip else g, e.t() if flip else e, "db" if flip else "da")


def _offsets(g, R, T, tail):
    cuts = torch.randint(0, T - tail + 1, (R + 1,), generator=g).sort().values
    return cuts.to(torch.int32).to(DEV)


CASES = [
    # R, T, K, N, r, n, dtype, ragged
    (1, 1, 8, 8, 1, 1, B16, False),
    (1, 1, 3840, 640, 16, 3, B16, False),
    (5, 5, 256, 1000, 16, 5, B16, False),
    (64, 64, 130, 96, 8, 7, B16, False),
    (130, 130, 64, 72, 4, 200, B16, False),
    (3, 96, 192, 320, 16, 2, B16, False),
    (2, 130, 64, 33, 32, 2, B16, False),
    (7, 333, 257, 1001, 12, 3, B16, True),
    (7, 333, 1001, 257, 12, 3, F32, True),
    (66, 500, 72, 65, 24, 9, B16, True),
    (4, 1000, 320, 192, 64, 4, B16, True),
    (3, 700, 96, 200, 128, 2, B16, True),
    (2, 301, 67, 61, 127, 3, F32, True),
    (3, 260, 50, 1, 80, 2, B16, True),
    (1, 77, 1, 40, 5, 1, B16, False),
    (9, 20, 1000, 1100, 16, 4, B16, True),    # up to four tokens to a request, one launch
    (40, 120, 515, 520, 64, 9, F32, False),
    (17, 17, 515, 600, 50, 9, B16, False),
    (12, 40, 136, 700, 33, 5, B16, True),
    (3, 2000, 1088, 72, 16, 2, B16, True),    # whole lines through LDS: one, two and more blocks of ranks
    (3, 2000, 520, 200, 24, 2, B16, True),
    (2, 1700, 72, 456, 72, 2, F32, True),
    (2, 8192, 40, 136, 120, 2, B16, False),
    (6, 4100, 160, 128, 40, 3, B16, True),   # blocks that share K between four waves
    (6, 9000, 64, 96, 96, 3, F32, True),
    (5, 8192, 128, 64, 16, 2, B16, True),
    (3, 8300, 136, 72, 16, 2, B16, True),    # tiles of 64 tokens
    (2, 8450, 72, 65, 24, 2, B16, False),
    (61, 300, 64, 72, 16, 4, B16, True),     # segments found at once, and after one and two searches
    (62, 300, 64, 72, 16, 4, B16, True),
    (5000, 6001, 64, 72, 8, 7, B16, True),
    (40, 3000, 520, 1100, 24, 20, B16, True),   # gradients' blocks that share a CU: two and more of them
    (20, 2000, 520, 1100, 72, 20, B16, False),
    (64, 4000, 520, 1100, 16, 64, B16, True),
    (64, 3000, 260, 513, 64, 96, B16, True),
]


@pytest.mark.parametrize("R,T,K,N,r,n,dtype,ragged", CASES)
def test_forward_and_backward(R, T, K, N, r, n, dtype, ragged):
    g = _gen(R * T + K + N + r)
    low = _low(g, n, r, K, N)
    index = torch.randint(-1, n + 1, (R,), generator=g).to(torch.int64 if T % 2 else torch.int32).to(DEV)
    if R == 1:
        index.zero_()
    requests = harp_amd.AdapterRequests(index, _offsets(g, R, T, T // 16) if ragged else None)
    x, base = _rand(g, T, K), _rand(g, T, N, dtype=dtype)
    out = harp_amd.add_adapters(base, x, low, requests)
    assert out.dtype == dtype and out.shape == base.shape
    _check(base, x, low, requests, out)
    if dtype == F32:
        return
    leaves = [t.requires_grad_() for t in (base, x, low.a, low.b)]
    out = harp_amd.add_adapters(base, x, low, requests)
    dy = _rand(g, T, N)
    gbase, *grads = torch.autograd.grad(out, leaves, dy)
    assert torch.equal(gbase, dy)
    _check(base, x, low, requests, out, dy, grads)


def test_tokens_without_an_adapter_keep_the_projection():
    g = _gen(2)
    low = _low(g, 2, 16, 64, 96)
    T = 150
    x, base = _rand(g, T, 64), _rand(g, T, 96)
    requests = harp_amd.AdapterRequests(torch.tensor([0, -1, 5, 1], device=DEV), torch.tensor([10, 40, 70, 90, 130], device=DEV))
    out = harp_amd.add_adapters(base, x, low, requests)
    for b, e, same in ((0, 10, True), (10, 40, False), (40, 90, True), (90, 130, False), (130, 150, True)):
        assert torch.equal(out[b:e], base[b:e]) == same
    # offsets outside the tokens are read as the nearest of them
    wide = harp_amd.AdapterRequests(requests.index, torch.tensor([-7, 40, 70, 90, 4000], device=DEV))
    _check(base, x, low, wide, harp_amd.add_adapters(base, x, low, wide))


def test_an_adapter_without_a_token_has_a_zero_gradient():
    g = _gen(4)
    low = _low(g, 5, 16, 64, 96)
    x, base = _rand(g, 64, 64), _rand(g, 64, 96)
    low.a.requires_grad_(), low.b.requires_grad_()
    requests = harp_amd.AdapterRequests(torch.tensor([3, 3], dtype=torch.int32, device=DEV))
    out = harp_amd.add_adapters(base, x, low, requests)
    ga, gb = torch.autograd.grad(out, (low.a, low.b), _rand(g, 64, 96))
    for i in range(5):
        assert bool((ga[i] == 0).all()) == (i != 3) and bool((gb[i] == 0).all()) == (i != 3)


def test_a_token_does_not_depend_on_the_batch():
    """The same token alone and among others, where both calls are small enough for 16 waves to share K: the same bits."""
    g = _gen(6)
    low = _low(g, 4, 16, 320, 192)
    x, base = _rand(g, 40, 320), _rand(g, 40, 192)
    index = torch.arange(40, device=DEV) % 4
    each = harp_amd.add_adapters(base, x, low, harp_amd.AdapterRequests(index))
    for i in (0, 7, 39):
        one = harp_amd.add_adapters(base[i:i + 1], x[i:i + 1], low, harp_amd.AdapterRequests(index[i:i + 1]))
        assert torch.equal(one[0], each[i])


@pytest.mark.parametrize("kind", ["batch", "padded", "odd", "strided", "expanded", "negated"])
def test_layouts(kind):
    g = _gen(8)
    low = _low(g, 2, 16, 72, 104)
    B, S = 2, 45
    x, base, dy = _rand(g, B, S, 72), _rand(g, B, S, 104), _rand(g, B, S, 104)
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))

    def view(t):
        if kind == "padded":
            return torch.cat((t, t), -1)[..., :t.size(-1)]
        if kind == "odd":
            return torch.cat((t[..., :1], t), -1)[..., 1:]
        if kind == "strided":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        if kind == "expanded":
            return t[:, :1].expand(-1, S, -1)
        if kind == "negated":
            return torch._neg_view(-t)
        return t

    if kind == "expanded":
        x, base, dy = (t[:, :1].repeat(1, S, 1) for t in (x, base, dy))
    results = []
    for f in (lambda t: t, view):
        xs, bs = f(x), f(base)
        if kind != "negated":
            xs = xs.detach().requires_grad_()
        a, b = (t.detach().clone().requires_grad_() for t in low[:2])
        out = harp_amd.add_adapters(bs, xs, harp_amd.Adapters(a, b, low.scales), requests)
        wrt = (a, b) + ((xs,) if kind != "negated" else ())
        results.append((out.detach(), *torch.autograd.grad(out, wrt, f(dy))))
    for p, q in zip(*results):
        assert torch.equal(p, q)
    if kind == "strided":  # a and b in another order
        other = harp_amd.Adapters(low.a.transpose(1, 2).contiguous().transpose(1, 2),
                                  low.b.transpose(0, 1).contiguous().transpose(0, 1), low.scales)
        assert torch.equal(harp_amd.add_adapters(base, x, other, requests), results[0][0])


def test_values_that_are_not_finite_stay_with_their_request():
    g = _gen(12)
    low = _low(g, 3, 16, 64, 96)
    with torch.no_grad():
        low.a[1] = float("nan")
        low.b[1] = float("inf")
    x, base = _rand(g, 48, 64), _rand(g, 48, 96)
    requests = harp_amd.AdapterRequests(torch.tensor([0, 1, 2], device=DEV))
    low.a.requires_grad_(), low.b.requires_grad_(), x.requires_grad_()
    out = harp_amd.add_adapters(base, x, low, requests)
    gx, ga, gb = torch.autograd.grad(out, (x, low.a, low.b), _rand(g, 48, 96))
    assert bool(out[16:32].isnan().all()) and bool(out[:16].isfinite().all()) and bool(out[32:].isfinite().all())
    for t in (ga, gb):
        assert bool(t[0].isfinite().all()) and bool(t[2].isfinite().all())
    assert bool(gx[:16].isfinite().all()) and bool(gx[32:].isfinite().all())


def test_no_tokens():
    g = _gen(14)
    low = _low(g, 2, 8, 16, 24)
    x = torch.zeros(0, 16, dtype=B16, device=DEV, requires_grad=True)
    base = torch.zeros(0, 24, dtype=B16, device=DEV)
    low.a.requires_grad_(), low.b.requires_grad_()
    out = harp_amd.add_adapters(base, x, low, harp_amd.AdapterRequests(torch.tensor([0, 1], device=DEV)))
    ga, gb, gx = torch.autograd.grad(out, (low.a, low.b, x), torch.zeros_like(out))
    assert out.shape == (0, 24) and bool((ga == 0).all()) and bool((gb == 0).all()) and gx.shape == x.shape


def test_gradients_of_some_only():
    g = _gen(16)
    low = _low(g, 2, 16, 64, 96)
    x, base, dy = _rand(g, 64, 64), _rand(g, 64, 96), _rand(g, 64, 96)
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
    full = None
    for want in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(w)) for t, w in zip((x, low.a, low.b), want)]
        out = harp_amd.add_adapters(base, leaves[0], harp_amd.Adapters(leaves[1], leaves[2], low.scales), requests)
        got = iter(torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dy))
        got = [next(got) if w else None for w in want]
        if full is None:
            full = got
        for a, b in zip(full, got):
            assert b is None or torch.equal(a, b)


def test_gradient_against_differences():
    """d out along a direction, in bf16 results of fp32 sums: the directional derivative of A by the
    difference of two fp32 results, exact up to 2^-22 of the terms, since out is linear in A."""
    g = _gen(18)
    low = _low(g, 2, 16, 64, 96)
    x, base, dy = _rand(g, 64, 64), torch.zeros(64, 96, device=DEV), _rand(g, 64, 96)
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
    leaves = [t.detach().requires_grad_() for t in (x, low.a, low.b)]
    out = harp_amd.add_adapters(base.to(B16), leaves[0], harp_amd.Adapters(leaves[1], leaves[2], low.scales), requests)
    grads = torch.autograd.grad(out, leaves, dy)
    for i, got in enumerate(grads):
        v = _rand(g, *got.shape, scale=0.1)
        args = [x, low.a, low.b]
        plus, minus = list(args), list(args)
        plus[i], minus[i] = (args[i].float() + v.float()).to(B16), (args[i].float() - v.float()).to(B16)
        moved = (plus[i].double() - minus[i].double())
        f = [harp_amd.add_adapters(base, a[0], harp_amd.Adapters(a[1], a[2], low.scales), requests).double()
             for a in (plus, minus)]
        diff = float(((f[0] - f[1]) * dy.double()).sum())
        along = got.double() * moved
        # each entry of the gradient is rounded once (2^-8)
        assert abs(diff - float(along.sum())) <= 2.0 ** -8 * float(along.abs().sum()) + 1e-3


def test_refusals():
    g = _gen(20)
    low = _low(g, 2, 16, 64, 96)
    x, base = _rand(g, 6, 64), _rand(g, 6, 96)
    ids = torch.tensor([0, 1], device=DEV)
    ok = harp_amd.AdapterRequests(ids)
    A, R = harp_amd.Adapters, harp_amd.AdapterRequests
    f = harp_amd.add_adapters
    for args, msg in [
        ((base, x.float(), low, ok), "x must be bfloat16"),
        ((base.half(), x, low, ok), "bfloat16 or float32"),
        ((base[:, :95], x, low, ok), "base must be"),
        ((base[:5], x, low, ok), "base must be"),
        ((base, x, A(low.a.float(), low.b), ok), "a must be a bfloat16"),
        ((base, x, A(low.a[:, :, :63], low.b), ok), "a must be"),
        ((base, x, A(low.a[:1], low.b), ok), "b must be"),
        ((base, x, A(low.a, low.b[:, :, :8]), ok), "b must be"),
        ((base, x, A(low.a, low.b, low.scales.double()), ok), "scales must be float32"),
        ((base, x, A(low.a, low.b, low.scales[:1]), ok), "scales must be float32"),
        ((base, x, low, R(ids.float())), "int32 or int64"),
        ((base, x, low, R(ids[None])), "vector"),
        ((base, x, low, R(ids[:0])), "at least one"),
        ((base, x, low, R(torch.zeros(4, dtype=torch.int32, device=DEV))), "requests of one length"),
        ((base, x, low, R(ids, ids)), "offsets must be 3 values"),
        ((base, x, low, R(ids.cpu())), "index must be on"),
        ((base, x, A(_rand(g, 1, 129, 64), _rand(g, 1, 96, 129)), ok), "1 to 128"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            f(*args)
    low.a.requires_grad_()
    with pytest.raises(RuntimeError, match="gradients need a bfloat16 base"):
        f(base.float(), x, low, ok)
    with pytest.raises(RuntimeError, match="scales has no gradient"):
        f(base, x, A(low.a, low.b, low.scales.clone().requires_grad_()), ok)
    out = f(base, x, low, ok)
    ga, = torch.autograd.grad(out.float().sum(), low.a, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        ga.float().sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(base, torch.autograd.forward_ad.make_dual(x, x), low, ok)


def _same_where_not_finite(got, want, signs):
    """An infinite t stays an infinity of its sign.  An infinity in B may become NaN: t is taken apart into hi + lo,
    lo is zero or of either sign, and hi inf + lo inf is then NaN."""
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    if signs:
        for f in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(f(got), f(want)), f


@pytest.mark.parametrize("T,r,dtype", [(3, 16, B16), (9, 16, B16), (60, 16, B16), (60, 40, F32), (600, 32, B16), (600, 16, F32)])
def test_infinities_stay_with_their_request_and_stay_infinities(T, r, dtype):
    """Three requests; the second's adapter sums to infinities (in t, or in B), the others' rows are as without it."""
    g = _gen(T + r)
    K, N, n = 64, 96, 3
    base, x = _rand(g, T, N, dtype=dtype), _rand(g, T, K)
    low = _low(g, n, r, K, N)
    requests = harp_amd.AdapterRequests(torch.tensor([0, 1, 2], device=DEV))
    clean = harp_amd.add_adapters(base, x, low, requests)
    part = slice(T // 3, 2 * (T // 3))
    for which in ("a", "b", "nan"):
        a, b = low.a.clone(), low.b.clone()
        if which == "a":  # one rank's t is an infinity of x's sign; the other ranks add finite values
            a[1] = 0
            a[1, 0, 5] = float("inf")
            a[1, 0, :5] = a[1, 0, 6:] = 0
            b[1, :, 1:] = 0
            x = x.clone()
            x[part, 5] = torch.where(x[part, 5] == 0, torch.ones_like(x[part, 5]), x[part, 5])
        else:
            b[1, 7, 0] = float("inf") if which == "b" else float("nan")
        out = harp_amd.add_adapters(base, x, harp_amd.Adapters(a, b, low.scales), requests)
        t = low.scales[1].double() * (x[part].double() @ a[1].double().t())
        if which == "a":
            t = torch.where(torch.arange(r, device=DEV) == 0, t, 0.0)
        want = base[part].double() + t @ b[1].double().t()
        _same_where_not_finite(out[part].double(), want, which == "a")
        assert not bool(torch.isfinite(want).all())
        others = torch.ones(T, dtype=torch.bool, device=DEV)
        others[part] = False
        if which != "a":
            assert torch.equal(out[others], clean[others])
        assert bool(torch.isfinite(out[others]).all())
