"""GPU tests of the operators for requests of one batch as a program uses them:
the q/k/v producer with adapters inside and its separate parts, the attention
block, 8-bit projections, captured graphs, other streams, two calls at once."""

import threading
from types import SimpleNamespace

import pytest
import torch
from torch import nn

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, scale=1.0, dtype=B16):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _low(g, n, r, K, N, scales=True):
    s = (torch.rand(n, generator=g) + 0.5).to(DEV) if scales else None
    return harp_amd.Adapters(nn.Parameter(_rand(g, n, r, K, scale=K ** -0.5)),
                             nn.Parameter(_rand(g, n, N, r, scale=0.5 * r ** -0.5)), s)


class _Norm(nn.Module):
    def __init__(self, w):
        super().__init__()
        self.weight, self.eps = nn.Parameter(w), EPS


def _attention(g, dim, heads, d=128, bias=False):
    attn = nn.Module()
    attn.heads = heads
    for name, n_in, n_out in (("to_q", dim, heads * d), ("to_k", dim, heads * d), ("to_v", dim, heads * d),
                              ("out", heads * d, dim)):
        lin = nn.Linear(n_in, n_out, bias=bias, dtype=B16, device=DEV)
        with torch.no_grad():
            lin.weight.copy_(_rand(g, n_out, n_in, scale=n_in ** -0.5))
        lin.requires_grad_(False)
        setattr(attn, name, lin)
    attn.to_out = nn.ModuleList([attn.out, nn.Identity()])
    attn.norm_q, attn.norm_k = (_Norm((1 + 0.1 * torch.randn(d, generator=g)).to(B16).to(DEV)) for _ in range(2))
    return attn


def _positions(g, B, S, rope):
    p = torch.randint(0, 300, (B, S, len(rope.axes_dims)), generator=g).to(torch.int32).to(DEV)
    return harp_amd.AxialPositions(p, rope)


ROPE = harp_amd.AxialRope((32, 48, 48), 256.0)


def _turn64(x, positions, rope):
    ang = torch.cat([positions[..., a, None].double() * theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
                     for a, (d, theta) in enumerate(zip(rope.axes_dims, rope.theta))], -1)[:, None]
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = (x[..., 0::2], x[..., 1::2]) if rope.layout == "interleaved" else x.chunk(2, -1)
    y = torch.stack((a * c - b * s, a * s + b * c), -1)
    return y.flatten(-2) if rope.layout == "interleaved" else y.transpose(-1, -2).flatten(-2)


def _qkv64(attn, x, positions, requests, leaves):
    """q, k, v in 64 bits; leaves: x, then (a, b) of q, k, v, then the norm weights, as doubles."""
    x = leaves[0]
    B, S, _ = x.shape
    flat = x.flatten(0, 1)
    index = requests.index.tolist()
    T = B * S
    offsets = [i * (T // len(index)) for i in range(len(index) + 1)] if requests.offsets is None else requests.offsets.tolist()
    out = []
    for i, m in enumerate((attn.to_q, attn.to_k, attn.to_v)):
        a, b = leaves[1 + 2 * i], leaves[2 + 2 * i]
        y = flat @ m.base.weight.double().t()
        delta = [y.new_zeros(offsets[0], y.size(1))]
        for j, which in enumerate(index):
            rows = flat[offsets[j]:offsets[j + 1]]
            if 0 <= which < a.size(0):
                sc = 1.0 if m.scales is None else float(m.scales[which])
                delta.append(sc * (rows @ a[which].t()) @ b[which].t())
            else:
                delta.append(y.new_zeros(rows.size(0), y.size(1)))
        delta.append(y.new_zeros(T - offsets[-1], y.size(1)))
        y = (y + torch.cat(delta)).view(B, S, attn.heads, -1).transpose(1, 2)
        if i < 2:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * leaves[7 + i]
            y = _turn64(y, positions.positions, positions.rope)
        out.append(y)
    return out


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm())


QKV = [
    # B, S, heads, dim, rank, adapters, requests' offsets
    (1, 96, 1, 64, 8, 1, None),
    (3, 50, 3, 192, 16, 2, None),
    (1, 300, 2, 128, 24, 3, [0, 3, 3, 150, 290]),
    (2, 200, 5, 320, 64, 4, [10, 130, 131, 260, 399]),
    (1, 1500, 2, 128, 128, 2, [0, 700, 1400]),
    (4, 1, 2, 128, 16, 4, None),
    (1, 5000, 10, 64, 16, 2, [0, 1, 2, 3, 4000, 5000]),     # the large blocks
    (3, 235, 30, 128, 72, 3, None),                         # whole blocks, a third of the CUs without one
    (1, 4300, 30, 128, 40, 3, [0, 2200, 4300]),             # and the second launch of smaller ones
]


@pytest.mark.parametrize("B,S,heads,dim,r,n,offsets", QKV)
def test_qkv_with_adapters(B, S, heads, dim, r, n, offsets):
    """One rounding behind 32-bit sums: on the average half of 2^-8 / sqrt(3) (0.11%) of a value and
    at most 2^-8 (0.39%), so 0.25% of the norm; a gradient passes through one rounded tensor
    more (the products' gradients, which library products read): 0.35%."""
    g = _gen(S + dim)
    attn = _attention(g, dim, heads)
    attn = harp_amd.adapt_attention(attn, **{t: _low(g, n, r, dim, heads * 128, t != "to_k") for t in ("to_q", "to_k", "to_v")})
    x = _rand(g, B, S, dim).requires_grad_()
    pos = _positions(g, B, S, ROPE)
    R = B if offsets is None else len(offsets) - 1
    index = (torch.arange(R, device=DEV) * 2 + 1) % (n + 1)  # one that is n takes none
    requests = harp_amd.AdapterRequests(index, None if offsets is None else torch.tensor(offsets, device=DEV))
    with torch.no_grad():
        served = harp_amd.project_qkv(attn, x, pos, requests=requests)
        tabled = harp_amd.project_qkv(attn, x, pos.table(), requests=requests)
    out = harp_amd.project_qkv(attn, x, pos, requests=requests)
    for a, b, c in zip(served, tabled, out):
        assert torch.equal(a, b) and torch.equal(a, c.detach())
        assert a.stride() == (S * heads * 128, 128, heads * 128, 1)
    params = [t for m in (attn.to_q, attn.to_k, attn.to_v) for t in (m.a, m.b)] + [attn.norm_q.weight, attn.norm_k.weight]
    leaves = [t.detach().double().requires_grad_() for t in [x] + params]
    want = _qkv64(attn, x, pos, requests, leaves)
    d = [_rand(g, B, S, heads, 128).transpose(1, 2) for _ in range(3)]
    grads = torch.autograd.grad(out, [x] + params, d)
    grads64 = torch.autograd.grad(want, leaves, [t.double() for t in d], materialize_grads=True)
    for a, b in zip(out, want):
        assert _rel(a.detach(), b.detach()) <= 2.5e-3
        assert float(((a.detach().double() - b.detach()).abs() / (b.detach().abs() + b.detach().abs().mean())).max()) <= 2.0 ** -7
    for i, (a, b) in enumerate(zip(grads, grads64)):
        if float(b.norm()) == 0:
            assert not bool(a.any())
        else:
            assert _rel(a, b) <= 3.5e-3, (i, _rel(a, b))


@pytest.mark.parametrize("B,S,heads,dim", [(3, 40, 2, 128), (1, 1, 3, 64), (2, 300, 2, 64), (2, 3000, 2, 64)])
def test_the_one_launch_takes_positions_of_all_or_of_each(B, S, heads, dim):
    """Positions of the whole batch, of each sample, as columns of a longer array, and their table: one result."""
    g = _gen(B * S)
    attn = harp_amd.adapt_attention(_attention(g, dim, heads), **{t: _low(g, 2, 16, dim, heads * 128) for t in ("to_q", "to_k", "to_v")})
    x = _rand(g, B, S, dim)
    requests = harp_amd.AdapterRequests(torch.arange(B, device=DEV) % 2)
    for dtype in (torch.int32, torch.int64, torch.float32):
        wide = torch.randint(0, 300, (S, 5), generator=g).to(dtype).to(DEV)
        p = wide[:, 1:4]
        forms = [p, p.contiguous()[None], p.expand(B, S, 3), p.expand(B, S, 3).contiguous(), wide.t().contiguous().t()[:, 1:4]]
        with torch.no_grad():
            want = harp_amd.project_qkv(attn, x, ROPE.table(p), requests=requests)
            for f in forms:
                for a, b in zip(harp_amd.project_qkv(attn, x, harp_amd.AxialPositions(f, ROPE), requests=requests), want):
                    assert torch.equal(a, b)


def test_qkv_without_the_one_launch():
    """The separate parts (here for pairs of the other layout, a bias, heads of 64, few-token requests) agree
    with 64 bits within a rounding of each part: three of 2^-8 / sqrt(3) at most, under 0.6%."""
    for d, layout, bias, ranks in ((128, "half", False, (16,) * 3), (64, "interleaved", True, (16,) * 3), (128, "interleaved", False, (16, 8, 12))):
        g = _gen(d)
        heads, dim, B, S = 2, 192, 3, 40
        attn = _attention(g, dim, heads, d, bias)
        if bias:
            for m in (attn.to_q, attn.to_k, attn.to_v):
                m.bias.data.zero_()
        rope = harp_amd.AxialRope((d // 4, d // 4, d // 2), 256.0, layout)
        attn = harp_amd.adapt_attention(attn, **{t: _low(g, 3, r, dim, heads * d) for t, r in zip(("to_q", "to_k", "to_v"), ranks)})
        x = _rand(g, B, S, dim).requires_grad_()
        pos = _positions(g, B, S, rope)
        requests = harp_amd.AdapterRequests(torch.tensor([2, 0, 1], device=DEV))
        out = harp_amd.project_qkv(attn, x, pos, requests=requests)
        params = [t for m in (attn.to_q, attn.to_k, attn.to_v) for t in (m.a, m.b)] + [attn.norm_q.weight, attn.norm_k.weight]
        leaves = [t.detach().double().requires_grad_() for t in [x] + params]
        want = _qkv64(attn, x, pos, requests, leaves)
        dy = [_rand(g, B, S, heads, d).transpose(1, 2) for _ in range(3)]
        grads = torch.autograd.grad(out, [x] + params, dy)
        grads64 = torch.autograd.grad(want, leaves, [t.double() for t in dy])
        for a, b in zip((*out, *grads), (*want, *grads64)):
            assert _rel(a.detach(), b.detach()) <= 6e-3


def test_one_launch_and_its_parts_agree():
    g = _gen(31)
    attn = harp_amd.adapt_attention(_attention(g, 192, 2), **{t: _low(g, 2, 16, 192, 256) for t in ("to_q", "to_k", "to_v")})
    x, pos = _rand(g, 2, 70, 192), _positions(g, 2, 70, ROPE)
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
    with torch.no_grad():
        one = harp_amd.project_qkv(attn, x, pos, requests=requests)
        parts = harp_amd.project_qkv(attn, x, pos, fused=False, requests=requests)
        bare = harp_amd.project_qkv(attn, x, pos)
        none = harp_amd.project_qkv(attn, x, pos, requests=harp_amd.AdapterRequests(torch.tensor([-1, 7], device=DEV)))
    for a, b, c, e in zip(one, parts, bare, none):
        assert _rel(a, b.double()) <= 6e-3 and _rel(e, c.double()) <= 6e-3 and _rel(a, c.double()) > 0.1


def test_attention_block_of_three_requests():
    """Projections with adapters, norm and rotation, ring attention and an adapted output projection: each
    request's rows are those of the same request alone."""
    g = _gen(37)
    dim, heads, S = 256, 2, 64
    attn = harp_amd.adapt_attention(_attention(g, dim, heads), **{t: _low(g, 4, 16, dim, dim) for t in ("to_q", "to_k", "to_v", "to_out")})
    block = harp_amd.RingZAttention(attn, 2)
    x, pos = _rand(g, 3, S, dim), _positions(g, 3, S, ROPE)
    index = torch.tensor([3, -1, 0], device=DEV)
    with torch.no_grad():
        all_ = block(x, pos, requests=harp_amd.AdapterRequests(index))
        for i in range(3):
            one = block(x[i:i + 1], harp_amd.AxialPositions(pos.positions[i:i + 1], ROPE),
                        requests=harp_amd.AdapterRequests(index[i:i + 1]))
            assert _rel(all_[i:i + 1], one.double()) <= 6e-3
    # trained: the adapters that were used get gradients
    out = block(x, pos, requests=harp_amd.AdapterRequests(index))
    out.float().square().sum().backward()
    for m in (attn.to_q, attn.to_k, attn.to_v, attn.to_out[0]):
        for t in (m.a, m.b):
            used = [bool(t.grad[i].any()) for i in range(4)]
            assert used == [True, False, False, True] and bool(t.grad.isfinite().all())


def test_8_bit_projections_with_adapters():
    """The 8-bit product and the adapters' part from the same tokens: the sum of both layers' results, one rounding apart."""
    g = _gen(41)
    lin = nn.Linear(192, 256, bias=False, dtype=B16, device=DEV).requires_grad_(False)
    for out_dtype in (B16, F32):
        base = harp_amd.Int8Linear.from_linear(lin, out_dtype)
        m = harp_amd.AdaptedLinear(base, _low(g, 2, 16, 192, 256))
        x = _rand(g, 2, 30, 192)
        requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
        with torch.no_grad():
            y = m(x, requests)
            assert y.dtype == out_dtype and torch.equal(m(x), base(x))
            want = base(x).double() + torch.stack([float(m.scales[i]) * x[j].double() @ m.a[i].double().t() @ m.b[i].double().t()
                                                  for j, i in enumerate((1, 0))])
            # bf16: half a step; fp32: 200 additions and what three bf16 leave of t
            assert _rel(y, want) <= (2.0 ** -8 if out_dtype == B16 else 1e-5)
            rows = harp_amd.quantize_int8(x)
            near = m(rows, requests)
            assert _rel(near, want) <= 2e-2  # the adapters see the 8-bit tokens
    attn = harp_amd.quantize_attention(_attention(g, 256, 2))
    attn = harp_amd.adapt_attention(attn, to_q=_low(g, 2, 8, 256, 256), to_v=_low(g, 2, 16, 256, 256))
    x, pos = _rand(g, 2, 48, 256), _positions(g, 2, 48, ROPE)
    requests = harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV))
    with torch.no_grad():
        q, k, v = harp_amd.project_qkv(attn, x, pos, requests=requests)
        rq, rk, rv = harp_amd.project_qkv(attn, harp_amd.quantize_int8(x), pos, requests=requests)
        _, k0, _ = harp_amd.project_qkv(attn, x, pos)
        assert torch.equal(k, k0) and torch.equal(k, rk) and _rel(q, rq.double()) <= 2e-2 and _rel(v, rv.double()) <= 2e-2
        out = harp_amd.RingZAttention(attn, 1)(x, pos, requests=requests)
        assert bool(out.isfinite().all())
    with pytest.raises(ValueError, match="8-bit hidden states"):
        mixed = harp_amd.adapt_attention(_attention(g, 256, 2), to_q=_low(g, 2, 8, 256, 256))
        harp_amd.project_qkv(mixed, harp_amd.quantize_int8(x), pos, requests=requests)


def test_positions_in_the_plain_projections():
    """Positions in the table's place: the one-launch producers read their table."""
    g = _gen(43)
    attn = _attention(g, 192, 2)
    x, pos = _rand(g, 2, 33, 192), _positions(g, 2, 33, ROPE)
    with torch.no_grad():
        for module in (attn, harp_amd.quantize_attention(attn)):
            for a, b in zip(harp_amd.project_qkv(module, x, pos), harp_amd.project_qkv(module, x, pos.table())):
                assert torch.equal(a, b)
        for a, b in zip(harp_amd.project_qkv(attn, x, pos, fused=False), harp_amd.project_qkv(attn, x, pos)):
            assert _rel(a, b.double()) <= 1e-2  # truncated there, rounded here
    half = harp_amd.AxialPositions(pos.positions, harp_amd.AxialRope((32, 48, 48), 256.0, "half"))
    xg = x.clone().requires_grad_()
    q, k, _ = harp_amd.project_qkv(attn, xg, half)
    gx, gw = torch.autograd.grad((q, k), (xg, attn.norm_q.weight), (torch.ones_like(q), torch.ones_like(k)))
    assert bool(gx.isfinite().all()) and bool(gw.any())


def _training_step(attn, x, pos, requests, d, base, low, dy):
    """q, k, v with their gradients, and a Linear's adapters with theirs."""
    qkv = harp_amd.project_qkv(attn, x, pos, requests=requests)
    leaves = [x] + [t for m in (attn.to_q, attn.to_k, attn.to_v) for t in (m.a, m.b)]
    grads = torch.autograd.grad(qkv, leaves, d)
    y = harp_amd.add_adapters(base, x, low, requests)
    more = torch.autograd.grad(y, (low.a, low.b), dy)
    q, k = harp_amd.qk_norm_axial_rope(qkv[0].detach().requires_grad_(), qkv[1].detach(), pos.positions, pos.rope,
                                       attn.norm_q.weight, None, EPS)
    last = torch.autograd.grad(q, attn.norm_q.weight, d[0])
    return [t.detach() for t in (*qkv, y, q, k, *grads, *more, *last)]


def _step_inputs(seed):
    g = _gen(seed)
    attn = harp_amd.adapt_attention(_attention(g, 192, 2), **{t: _low(g, 3, 16, 192, 256) for t in ("to_q", "to_k", "to_v")})
    x = _rand(g, 2, 90, 192).requires_grad_()
    return (attn, x, _positions(g, 2, 90, ROPE), harp_amd.AdapterRequests(torch.tensor([2, 0], device=DEV)),
            [_rand(g, 2, 90, 2, 128).transpose(1, 2) for _ in range(3)], _rand(g, 2, 90, 100), _low(g, 3, 32, 192, 100),
            _rand(g, 2, 90, 100))


def test_graph_capture_and_replay():
    """A captured step, replayed with other adapters, tokens and positions between eager steps: the eager results."""
    args = _step_inputs(47)
    attn, x, pos, requests = args[:4]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _training_step(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _training_step(*args)
    for i in range(4):
        with torch.no_grad():
            x.copy_(_rand(_gen(100 + i), *x.shape))
            requests.index.copy_(torch.tensor([i % 3, (i + 1) % 4], device=DEV))
            pos.positions.copy_(pos.positions + i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = _training_step(*args)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_captured_graphs_and_a_capture_beside_a_live_graph():
    a, b = _step_inputs(53), _step_inputs(59)
    graphs = []
    for args in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _training_step(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, _training_step(*args), args))
    for _ in range(3):
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out, args in graphs:
            for p, q in zip(out, _training_step(*args)):
                assert torch.equal(p, q)
    # leaves of a live eager graph of another stream: refused, not the end of the process
    attn, x, pos, requests = a[:4]
    low, base = a[6], a[5]
    live = (harp_amd.project_qkv(attn, x, pos, requests=requests), harp_amd.add_adapters(base, x, low, requests),
            harp_amd.qk_norm_axial_rope(x.unflatten(-1, (-1, 64)).transpose(1, 2)[..., :64], None, pos.positions,
                                        harp_amd.AxialRope((16, 24, 24), 256.0), None, None, EPS))
    calls = (lambda: harp_amd.project_qkv(attn, x, pos, requests=requests),
             lambda: harp_amd.add_adapters(base, x, low, requests),
             lambda: harp_amd.qk_norm_axial_rope(x.view(2, 90, 3, 64).detach().transpose(1, 2), None, pos.positions,
                                                 harp_amd.AxialRope((16, 24, 24), 256.0), attn_w, None, EPS))
    attn_w = torch.ones(64, device=DEV, requires_grad=True)
    live += (harp_amd.qk_norm_axial_rope(x.view(2, 90, 3, 64).detach().transpose(1, 2), None, pos.positions,
                                         harp_amd.AxialRope((16, 24, 24), 256.0), attn_w, None, EPS),)
    for call in calls:
        with pytest.raises(RuntimeError, match="live autograd graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del live


def test_other_streams_and_threads():
    """Two threads with a stream each, both kinds of calls at once: the results of the default stream."""
    inputs = [_step_inputs(61 + i) for i in range(2)]
    want = [_training_step(*a) for a in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = _training_step(*inputs[i])
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_training_step_of_a_linear_with_adapters():
    """AdaptedLinear in a step of an optimiser: the base stays, the adapters of the batch's requests move."""
    g = _gen(67)
    m = harp_amd.AdaptedLinear(nn.Linear(64, 96, dtype=B16, device=DEV).requires_grad_(False), _low(g, 3, 8, 64, 96))
    before = {k: v.clone() for k, v in m.state_dict().items()}
    opt = torch.optim.SGD([m.a, m.b], lr=0.1)
    x = _rand(g, 2, 20, 64)
    y = m(x, harp_amd.AdapterRequests(torch.tensor([2, 0], device=DEV)))
    y.float().square().sum().backward()
    opt.step()
    for k, v in m.state_dict().items():
        if k in ("a", "b"):
            assert [not torch.equal(v[i], before[k][i]) for i in range(3)] == [True, False, True]
        else:
            assert torch.equal(v, before[k])


def test_refusals():
    g = _gen(71)
    attn = harp_amd.adapt_attention(_attention(g, 128, 1), **{t: _low(g, 2, 16, 128, 128) for t in ("to_q", "to_k", "to_v")})
    x, pos = _rand(g, 2, 8, 128), _positions(g, 2, 8, ROPE)
    ok = harp_amd.AdapterRequests(torch.tensor([0, 1], device=DEV))
    with pytest.raises(RuntimeError, match="positions must be"):
        harp_amd.project_qkv(attn, x, harp_amd.AxialPositions(pos.positions[:, :5], ROPE), requests=ok)
    with pytest.raises(RuntimeError, match="requests of one length"):
        harp_amd.project_qkv(attn, x, pos, requests=harp_amd.AdapterRequests(torch.zeros(3, dtype=torch.int32, device=DEV)))
    with pytest.raises(ValueError, match="adapt_attention"):
        harp_amd.project_qkv(_attention(g, 128, 1), x, pos, requests=ok)
    out = harp_amd.project_qkv(attn, x, pos, requests=ok)
    ga, = torch.autograd.grad(out[0].float().sum(), attn.to_q.a, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        ga.float().sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            harp_amd.project_qkv(attn, torch.autograd.forward_ad.make_dual(x, x), pos, requests=ok)
    empty = harp_amd.project_qkv(attn, x[:, :0].requires_grad_(), harp_amd.AxialPositions(pos.positions[:, :0], ROPE), requests=ok)
    assert all(t.shape == (2, 1, 0, 128) for t in empty)
    ga, = torch.autograd.grad(empty[0].float().sum(), attn.to_q.a)
    assert not bool(ga.any())


def test_a_weight_shared_by_two_captured_calls():
    """One leaf in two calls of one capture, the first one's graph alive: both are of the capture's own stream."""
    g = _gen(73)
    x, res = _rand(g, 6, 64).requires_grad_(), _rand(g, 6, 64)
    w = torch.ones(64, dtype=B16, device=DEV, requires_grad=True)
    d = _rand(g, 6, 64)

    def step():
        y, h = harp_amd.add_rms_norm(x, res, w, EPS)
        z, _ = harp_amd.add_rms_norm(y, h, w, EPS)
        return torch.autograd.grad(z, (x, w), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_a_broken_adapter_stays_with_its_request():
    """Infinities and NaN in one adapter's B reach no token of the requests in the same block of the one launch."""
    for r, S, heads in ((16, 24, 2), (72, 40, 2), (16, 900, 30)):
        g = _gen(r + S)
        attn = harp_amd.adapt_attention(_attention(g, 128, heads), **{t: _low(g, 3, r, 128, heads * 128) for t in ("to_q", "to_k", "to_v")})
        x, pos = _rand(g, 3, S, 128), _positions(g, 3, S, ROPE)
        for index in ([0, 1, 2], [2, 1, -1], [1, 0, 5]):
            requests = harp_amd.AdapterRequests(torch.tensor(index, device=DEV))
            with torch.no_grad():
                clean = harp_amd.project_qkv(attn, x, pos, requests=requests)
                kept = [m.b.clone() for m in (attn.to_q, attn.to_k, attn.to_v)]
                for m in (attn.to_q, attn.to_k, attn.to_v):
                    m.b[1, 3::7] = float("inf")
                    m.b[1, 4::9, 0] = float("nan")
                broken = harp_amd.project_qkv(attn, x, pos, requests=requests)
                for m, b in zip((attn.to_q, attn.to_k, attn.to_v), kept):
                    m.b.copy_(b)
            for a, b in zip(broken, clean):
                for i, which in enumerate(index):
                    if which == 1:
                        assert not bool(torch.isfinite(a[i]).all())
                    else:
                        assert torch.equal(a[i], b[i])


@pytest.mark.parametrize("r", [8, 16, 128])
@pytest.mark.parametrize("form,norm", [("positions", True), ("table", True), ("table of each", True), ("none", True),
                                       ("none", False)])
def test_a_token_s_rounding_does_not_depend_on_the_batch(r, form, norm):
    """The same tokens with the same adapter, as two requests (one launch) and as 32 short ones (parts): both are one
    rounding of 32-bit sums, whose order differs by 2^-20 of a value and moves one of 2^9 results over a border
    between bf16 values (2^-6 leaves room for small ones); three roundings move every second."""
    g = _gen(r)
    attn = harp_amd.adapt_attention(_attention(g, 256, 3), **{t: _low(g, 3, r, 256, 384) for t in ("to_q", "to_k", "to_v")})
    if not norm:
        attn.norm_q = attn.norm_k = None
    B, S = 2, 48
    x = _rand(g, B, S, 256)
    pos = _positions(g, B, S, ROPE)
    freqs = {"positions": pos, "table": ROPE.table(pos.positions[0]), "table of each": pos.table(), "none": None}[form]
    cuts = torch.linspace(0, B * S, 33).round().to(torch.int32).to(DEV)
    two = harp_amd.AdapterRequests(torch.tensor([2, 2], device=DEV))
    many = harp_amd.AdapterRequests(torch.full((32,), 2, device=DEV), cuts)
    with torch.no_grad():
        want = harp_amd.project_qkv(attn, x, freqs, requests=two)
        got = harp_amd.project_qkv(attn, x, freqs, requests=many)
        each = harp_amd.project_qkv(attn, x, freqs, requests=harp_amd.AdapterRequests(torch.full((96,), 2, device=DEV)))
    for a, b, c in zip(want, got, each):
        assert a.stride() == b.stride() == (S * 384, 128, 384, 1) and b.dtype == B16
        for d in (b, c):
            assert float((a != d).float().mean()) <= 2.0 ** -6
            assert float(((a.double() - d.double()).abs() / (a.double().abs() + a.double().abs().mean())).max()) <= 2.0 ** -7
    if form == "positions":  # with a gradient: the one launch
        xg = x.clone().requires_grad_()
        for a, b in zip(want, harp_amd.project_qkv(attn, xg, freqs, requests=many)):
            assert torch.equal(a, b.detach())


def test_short_requests_in_a_captured_graph():
    g = _gen(71)
    attn = harp_amd.adapt_attention(_attention(g, 192, 2), **{t: _low(g, 5, 16, 192, 256) for t in ("to_q", "to_k", "to_v")})
    x, pos = _rand(g, 24, 1, 192), _positions(g, 24, 1, ROPE)
    index = torch.arange(24, device=DEV) % 6
    requests = harp_amd.AdapterRequests(index)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        for freqs in (pos, pos.table()):
            harp_amd.project_qkv(attn, x, freqs, requests=requests)
    torch.cuda.current_stream().wait_stream(side)
    for freqs in (pos, pos.table()):
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            out = harp_amd.project_qkv(attn, x, freqs, requests=requests)
        for k in range(3):
            x.copy_(_rand(g, 24, 1, 192))
            index.copy_((torch.arange(24, device=DEV) * (k + 1)) % 6)
            graph.replay()
            with torch.no_grad():
                want = harp_amd.project_qkv(attn, x, freqs, requests=requests)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_projections_without_a_token():
    """No sample, or samples without a token: empty q, k and v from every form of the projections, and gradients."""
    g = _gen(73)
    base = _attention(g, 192, 2)
    rows = harp_amd.quantize_attention(base)
    attn = harp_amd.adapt_attention(base, **{t: _low(g, 5, 16, 192, 256) for t in ("to_q", "to_k", "to_v")})
    low8 = harp_amd.adapt_attention(rows, to_q=_low(g, 5, 16, 192, 256))
    requests = harp_amd.AdapterRequests(torch.zeros(9, dtype=torch.int32, device=DEV))
    for B, S in ((0, 4), (2, 0)):
        x, pos = _rand(g, B, S, 192), _positions(g, B, S, ROPE)
        for freqs in (pos, pos.table(), None):
            calls = [(m, fused, None) for m in (base, rows, attn, low8) for fused in (True, False)]
            calls += [(m, fused, r) for m in (attn, low8) for fused in (True, False)
                      for r in (requests, harp_amd.AdapterRequests(requests.index[:1]))]
            for module, fused, r in calls:
                with torch.no_grad():
                    for t in harp_amd.project_qkv(module, x, freqs, fused=fused, requests=r):
                        assert t.shape == (B, 2, S, 128) and t.dtype == B16
                if module is base or module is attn:
                    leaves = [x.clone().requires_grad_(), base.norm_q.weight] + ([attn.to_q.a, attn.to_v.b] if r else [])
                    out = harp_amd.project_qkv(module, leaves[0], freqs, fused=fused, requests=r)
                    for a, t in zip(torch.autograd.grad(out, leaves, out, allow_unused=True), leaves):
                        assert a is None or (a.shape == t.shape and not bool(a.any()))


def test_an_adapted_module_without_requests_keeps_the_one_launch(monkeypatch):
    """No requests: with a table or no rotation the call of the module without adapters, bit for bit, with gradients
    too; with positions the call of requests that take none.  No separate projection runs."""
    g = _gen(79)
    base = _attention(g, 192, 2)
    names = ("to_q", "to_k", "to_v")
    x, pos = _rand(g, 2, 70, 192), _positions(g, 2, 70, ROPE)
    attn = harp_amd.adapt_attention(base, **{t: _low(g, 2, 16, 192, 256) for t in names})
    some = harp_amd.adapt_attention(base, to_q=_low(g, 2, 8, 192, 256), to_v=_low(g, 2, 16, 192, 256))

    def no_parts(*_):
        raise AssertionError("a projection of its own")

    for m in (base.to_q, base.to_k, base.to_v):
        monkeypatch.setattr(m, "forward", no_parts)
    with torch.no_grad():
        for freqs in (pos.table(), ROPE.table(pos.positions[0]), None):
            for module in (attn, some):
                for a, b in zip(harp_amd.project_qkv(module, x, freqs), harp_amd.project_qkv(base, x, freqs)):
                    assert torch.equal(a, b) and a.stride() == b.stride()
        nobody = harp_amd.AdapterRequests(torch.tensor([-1, 7], device=DEV))
        for a, b in zip(harp_amd.project_qkv(attn, x, pos), harp_amd.project_qkv(attn, x, pos, requests=nobody)):
            assert torch.equal(a, b)
    leaves = (x.requires_grad_(), base.norm_q.weight, base.norm_k.weight)
    d = [_rand(g, 2, 70, 2, 128).transpose(1, 2) for _ in range(3)]
    for freqs in (pos.table(), pos):
        out = harp_amd.project_qkv(attn, x, freqs)
        grads = torch.autograd.grad(out, leaves + (attn.to_q.a, attn.to_v.b), d, allow_unused=True)
        assert grads[3] is None and grads[4] is None  # the adapters take no part
        if freqs is pos:
            same = harp_amd.project_qkv(attn, x, pos, requests=nobody)
        else:
            same = harp_amd.project_qkv(base, x, freqs)
        for a, b in zip((*out, *grads[:3]), (*same, *torch.autograd.grad(same, leaves, d))):
            assert torch.equal(a, b)
    rows = harp_amd.quantize_attention(_attention(g, 192, 2))
    low8 = harp_amd.adapt_attention(rows, **{t: _low(g, 2, 16, 192, 256) for t in names})
    with torch.no_grad():
        for freqs in (pos.table(), None):
            for h in (x.detach(), harp_amd.quantize_int8(x.detach())):
                for a, b in zip(harp_amd.project_qkv(low8, h, freqs), harp_amd.project_qkv(rows, h, freqs)):
                    assert torch.equal(a, b)


def test_conjugated_and_negated_tables():
    """A table that is a lazy conjugate (the rotation back) or a negated view, in the one launch and in parts."""
    g = _gen(83)
    base = _attention(g, 192, 2)
    attn = harp_amd.adapt_attention(base, **{t: _low(g, 2, 16, 192, 256) for t in ("to_q", "to_k", "to_v")})
    rows = harp_amd.quantize_attention(base)
    x, pos = _rand(g, 2, 40, 192), _positions(g, 2, 40, ROPE)
    requests = [harp_amd.AdapterRequests(torch.tensor([1, 0], device=DEV)),
                harp_amd.AdapterRequests(torch.arange(16, device=DEV) % 2)]
    table = pos.table()
    for lazy in (table.conj(), torch._neg_view(table), torch._neg_view(table).conj()):
        plain = lazy.clone().resolve_conj().resolve_neg().contiguous()
        assert (lazy.is_conj() or lazy.is_neg()) and not (plain.is_conj() or plain.is_neg())
        calls = [lambda f: harp_amd.project_qkv(base, x, f), lambda f: harp_amd.project_qkv(rows, x, f),
                 lambda f: harp_amd.project_qkv(base, x, f, fused=False),
                 *(lambda f, r=r: harp_amd.project_qkv(attn, x, f, requests=r) for r in (None, *requests))]
        with torch.no_grad():
            for call in calls:
                for a, b in zip(call(lazy), call(plain)):
                    assert torch.equal(a, b)
        xg, grads = x.clone().requires_grad_(), []
        for f in (lazy, plain):
            out = harp_amd.project_qkv(base, xg, f)
            grads.append(torch.autograd.grad(out, xg, [torch.ones_like(t) for t in out])[0])
        assert torch.equal(*grads)


def test_a_table_with_a_gradient_is_refused_for_short_requests_too():
    g = _gen(89)
    base = _attention(g, 192, 2).requires_grad_(False)
    low = [harp_amd.Adapters(_rand(g, 2, 16, 192), _rand(g, 2, 256, 16)) for _ in range(3)]
    attn = harp_amd.adapt_attention(base, **dict(zip(("to_q", "to_k", "to_v"), low)))
    x, table = _rand(g, 1, 16, 192), _positions(g, 1, 16, ROPE).table().requires_grad_()
    for count in (1, 16):
        requests = harp_amd.AdapterRequests(torch.zeros(count, dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="rotation has no gradient"):
            harp_amd.project_qkv(attn, x, table, requests=requests)
