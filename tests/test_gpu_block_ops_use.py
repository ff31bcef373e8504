"""GPU tests of the operators around the attention block as a program uses
them: one after the other, captured into HIP graphs, on other streams, and in
the attention block."""

import math
import threading

import pytest
import torch
from torch import nn

import harp_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
B16 = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, scale=1.0, dtype=B16):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


class _Norm(nn.Module):
    def __init__(self, w):
        super().__init__()
        self.weight, self.eps = nn.Parameter(w), 1e-6


def _attention(g, dim, heads, d=128, bias=False):
    attn = nn.Module()
    attn.heads = heads
    for name, n_in, n_out in (("to_q", dim, heads * d), ("to_k", dim, heads * d), ("to_v", dim, heads * d),
                              ("out", heads * d, dim)):
        lin = nn.Linear(n_in, n_out, bias=bias, dtype=B16, device=DEV)
        with torch.no_grad():
            lin.weight.copy_(_rand(g, n_out, n_in, scale=n_in ** -0.5))
            if bias:
                lin.bias.copy_(_rand(g, n_out, scale=0.1))
        setattr(attn, name, lin)
    attn.to_out = nn.ModuleList([attn.out, nn.Identity()])
    attn.norm_q, attn.norm_k = (_Norm((1 + 0.1 * torch.randn(d, generator=g)).to(B16).to(DEV)) for _ in range(2))
    return attn


def _freqs(S, d=128):
    ang = torch.arange(S, dtype=torch.float64)[:, None] * (256.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    return torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(DEV)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _block(attn, x, res, w, freqs, sp=2):
    """One attention half of a transformer block in 8 bits: norm, attention, addition with the next norm."""
    rows, h = harp_amd.add_rms_norm_int8(x, res, w, 1e-5)
    out = harp_amd.RingZAttention(attn, sp)(rows, freqs)
    return harp_amd.add_rms_norm(out, h, w, 1e-5)


@pytest.mark.parametrize("S,heads,d,bias", [(64, 2, 128, False), (300, 3, 128, False), (128, 2, 64, False), (96, 2, 128, True)])
def test_attention_half_of_a_block(S, heads, d, bias):
    """The 8-bit block against its own stages in 64 bits: each stage's result
    is rounded to 8 or 16 bits, a relative step of 2^-8 or 1 / 127 of a row's
    maximum (about 4 standard deviations, so 1 / 127 * 4 / sqrt(12) = 0.9% of
    a value) per operand of the four products: under 4% of the result's norm."""
    g = _gen(S)
    dim = heads * d
    attn = _attention(g, dim, heads, d, bias)
    x, res, w = _rand(g, 1, S, dim), _rand(g, 1, S, dim, dtype=torch.float32), _rand(g, dim, scale=0.1) + 1
    f = _freqs(S, d)
    with torch.no_grad():
        q8 = harp_amd.quantize_attention(attn)
        y, h2 = _block(q8, x, res, w, f)
        h = (x.float() + res).double()
        n = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w.double()

        def lin(t, m):
            r = t @ m.weight.double().t()
            return r if m.bias is None else r + m.bias.double()

        def heads_of(t, norm):
            t = t.view(1, S, heads, d).transpose(1, 2)
            if norm is None:
                return t
            t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
            return torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (d // 2, 2)).contiguous())
                                      * f.to(torch.complex128)).flatten(-2)

        q, k, v = (heads_of(lin(n, m), nm) for m, nm in ((attn.to_q, attn.norm_q), (attn.to_k, attn.norm_k), (attn.to_v, None)))
        p = torch.softmax(torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d), -1)
        o = lin(torch.matmul(p, v.contiguous()).transpose(1, 2).reshape(1, S, dim), attn.out)
        want_h = h + o
        want = want_h / torch.sqrt(want_h.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    print(f"[block S={S} heads={heads} d={d} bias={bias}: rel {_rel(y, want):.2e}, out {_rel(h2.double() - h, o):.2e}]", flush=True)
    assert h2.dtype == torch.float32 and y.dtype == B16
    assert _rel(h2.double() - h, o) <= 0.04 and _rel(y, want) <= 0.04


def test_training_chain():
    """Two norms around a Linear, the residual stream passing both, against
    autograd on the formulas in 64 bits: bf16 roundings of the chain's values
    (2^-8 each, four stages) stay under 3% of a gradient's norm."""
    g = _gen(7)
    T, C = 200, 320
    x, res = _rand(g, T, C), _rand(g, T, C)
    w1, w2, m = _rand(g, C, scale=0.1) + 1, _rand(g, C, scale=0.1) + 1, _rand(g, C, C, scale=C ** -0.5)
    dy = _rand(g, T, C)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w1, w2, m)]
    a, r, u1, u2, mm = leaves
    y, h = harp_amd.add_rms_norm(a, r, u1)
    y2, h2 = harp_amd.add_rms_norm(y @ mm, h, u2)
    got = torch.autograd.grad((y2, h2), leaves, (dy, dy))
    leaves64 = [t.double().requires_grad_(True) for t in (x, res, w1, w2, m)]
    a, r, u1, u2, mm = leaves64

    def norm(t, w):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w

    h = a + r
    h2 = norm(h, u1) @ mm + h
    want = torch.autograd.grad((norm(h2, u2), h2), leaves64, (dy.double(), dy.double()))
    for p, q, name in zip(got, want, ("x", "res", "w1", "w2", "m")):
        assert _rel(p, q) <= 0.03, (name, _rel(p, q))


def _serve(layer, attn, x, res, w, f):
    with torch.no_grad():
        y, h = _block(attn, x, res, w, f)
        return layer(y), h


def _train(x, res, w, dy):
    y, h = harp_amd.add_rms_norm(x, res, w)
    return (y, h, *torch.autograd.grad((y, h), (x, res, w), (dy, dy)))


def test_graph_capture_and_replay():
    """Serving and training calls captured into one graph each, replayed with
    new inputs and the program's own work between: equal to the eager results,
    bit for bit, at every replay; two graphs share nothing."""
    g = _gen(3)
    dim = 256
    attn = harp_amd.quantize_attention(_attention(g, dim, 2))
    w = _rand(g, dim, scale=0.1) + 1
    f = _freqs(130)
    shapes = (130, 1)  # a prompt and a single token
    graphs = []
    for S in shapes:
        layer = harp_amd.Int8Linear.from_linear(nn.Linear(dim, 300, dtype=B16, device=DEV))
        x, res = _rand(g, 1, S, dim), _rand(g, 1, S, dim)
        t = [_rand(g, S, dim).requires_grad_(True) for _ in range(2)] + [w.clone().requires_grad_(True)]
        dy = _rand(g, S, dim)
        fr = f[:S]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                with torch.no_grad():
                    _block(attn, x, res, w, fr, 1), layer(x)
                _train(*t, dy)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with torch.no_grad():
                y, h = _block(attn, x, res, w, fr, 1)
                outs = [layer(y), h]
            outs += list(_train(*t, dy))
        graphs.append((graph, layer, x, res, t, dy, fr, outs))
    for i in range(4):
        for graph, layer, x, res, t, dy, fr, outs in graphs:
            with torch.no_grad():
                for a in (x, res, *t, dy):
                    a.copy_(torch.randn(a.shape, generator=g).to(a.dtype))
            graph.replay()
            got = [o.clone() for o in outs]
            with torch.no_grad():
                y, h = _block(attn, x, res, w, fr, 1)
                want = [layer(y), h]
            want += list(_train(*t, dy))
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), i


def test_capture_beside_a_live_eager_graph():
    """While an eager graph of the same leaves is alive, capturing a step of
    them raises (torch's engine would end the process in the backward);
    afterwards the eager graph's own backward still runs, and once it is gone
    the step is captured and replays equal to the eager one."""
    g = _gen(8)
    x, res = (_rand(g, 40, 96).requires_grad_(True) for _ in range(2))
    w = (_rand(g, 96, scale=0.1) + 1).requires_grad_(True)
    dy = _rand(g, 40, 96)
    want = [t.detach() for t in _train(x, res, w, dy)]
    y, h = harp_amd.add_rms_norm(x, res, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="live autograd graph"):
        with torch.cuda.graph(graph):
            harp_amd.add_rms_norm(x, res, w)
    torch.cuda.synchronize()
    got = torch.autograd.grad((y, h), (x, res, w), (dy, dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want[2:]))
    del y, h, got
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _train(x, res, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _train(x, res, w, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_streams_and_threads():
    """Calls at once on several streams, from several threads, each equal to
    its result alone."""
    g = _gen(9)
    layers, inputs, want = [], [], []
    for M, N, K in ((1, 700, 512), (200, 384, 640), (500, 1024, 256), (33, 200, 2000)):
        lin = nn.Linear(K, N, dtype=B16, device=DEV)
        layers.append(harp_amd.Int8Linear.from_linear(lin))
        inputs.append((_rand(g, M, K), (_rand(g, K, scale=0.1) + 1).requires_grad_(True), _rand(g, M, K)))
    def work(i):
        x, w, dy = inputs[i]
        with torch.no_grad():
            y = layers[i](x)
        n, _ = harp_amd.add_rms_norm(x, None, w)
        (gw,) = torch.autograd.grad(n, w, dy)
        return y, n.detach(), gw
    want = [work(i) for i in range(len(layers))]
    torch.cuda.synchronize()
    got = {}

    def thread(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = work(i)
        s.synchronize()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(layers))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(a, b) for a, b in zip(got[i], w)), i


def test_results_do_not_depend_on_what_else_is_in_the_batch():
    """A token's result is the same alone and among others, whatever kinds of
    blocks the two calls take: the sums are exact and the epilogue's order of
    operations is one."""
    g = _gen(10)
    layer = harp_amd.Int8Linear.from_linear(nn.Linear(300, 520, dtype=B16, device=DEV))
    x = _rand(g, 700, 300)
    with torch.no_grad():
        full = layer(x)
        for n in (1, 16, 17, 70, 256, 513):
            assert torch.equal(layer(x[:n]), full[:n]), n
            assert torch.equal(layer(x[700 - n:]), full[700 - n:]), n
        assert torch.equal(layer(x[5]), full[5])


def test_modules_round_trip():
    g = _gen(12)
    attn = _attention(g, 256, 2)
    q8 = harp_amd.quantize_attention(attn)
    rows = harp_amd.quantize_int8(attn.to_q.weight.detach())
    assert torch.equal(q8.to_q.weight.values, rows.values) and torch.equal(q8.to_q.weight.scales, rows.scales)
    assert q8.norm_q is attn.norm_q and q8.heads == 2
    x, f = _rand(g, 1, 64, 256), _freqs(64)
    with torch.no_grad():
        y = harp_amd.RingZAttention(q8, 2)(x, f)
        other = harp_amd.quantize_attention(_attention(_gen(13), 256, 2))
        other.load_state_dict(q8.state_dict())
        assert torch.equal(harp_amd.RingZAttention(other, 2)(x, f), y)
        # 8-bit rows in place of the tensor, and the same input quantised by the module
        assert torch.equal(harp_amd.RingZAttention(q8, 2)(harp_amd.quantize_int8(x), f), y)
    with pytest.raises(RuntimeError, match="forward only"):
        harp_amd.RingZAttention(q8, 2)(x.requires_grad_(True), f)
    with pytest.raises(RuntimeError, match="features"):
        q8.to_q(x.detach()[..., :128])
    with pytest.raises(ValueError, match="multiple of sp_size"):
        harp_amd.RingZAttention(q8, 3)(x.detach(), f)


@pytest.mark.parametrize("which", [("to_q",), ("to_v",), ("to_q", "to_k")], ids=str)
def test_some_projections_in_8_bits(which):
    """An Int8Linear stands in for any of the projections: they then run one by one."""
    attn = _attention(_gen(14), 256, 2)
    for name in which:
        setattr(attn, name, harp_amd.Int8Linear.from_linear(getattr(attn, name)))
    x, f = _rand(_gen(15), 1, 64, 256), _freqs(64)
    with torch.no_grad():
        for a, b in zip(harp_amd.project_qkv(attn, x, f), harp_amd.project_qkv(attn, x, f, fused=False)):
            assert a.shape == (1, 2, 64, 128) and torch.equal(a, b)
        assert torch.equal(harp_amd.project_qkv(attn, x, f)[2], attn.to_v(x).unflatten(-1, (2, 128)).transpose(1, 2))
        assert bool(torch.isfinite(harp_amd.RingZAttention(attn, 2)(x, f)).all())
        with pytest.raises(ValueError, match="8-bit projections"):
            harp_amd.project_qkv(attn, harp_amd.quantize_int8(x), f)
