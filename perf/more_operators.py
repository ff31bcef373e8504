"""Performance cases of the operators that give every request of a batch its own
positions and its own adapter: rotary positions with several axes, and low-rank
adapters beside a shared projection.

Every case is a plain dict; ``prepare`` makes what a user's program holds before
the call (inputs, adapters, modules), ``run`` is one pass, ``exact`` is the same
result in 64 bits.  Kinds:

* ``rope``: :func:`harp_amd.qk_norm_axial_rope`, the RMSNorm and the rotation of
  queries and keys from the positions of their tokens; forward, or forward +
  backward (``train``);
* ``adapters``: :func:`harp_amd.add_adapters`, a projection's result plus the
  low-rank adapter of each token's request; forward, or forward + backward;
* ``qkv``: :func:`harp_amd.project_qkv` on an attention module with adapters
  (:func:`harp_amd.adapt_attention`), the requests' positions in the place of
  the RoPE table; forward, or forward + backward with frozen projections.

With ``own`` false ``run`` computes the operators from elementary torch
operations in 32 bits (the angles in 64) instead.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
HEAD = 128
THETA = 256.0


def _rope(name, B, S, HQ, HK, D, train=False, norm=True, half=False, dtype="bf16", pos="int32", each=False):
    """B sequences of S tokens, HQ query and HK key heads of D features; ``half``: the pairs are (p, p + D/2);
    ``each``: every sequence has positions of its own."""
    case = {"kind": "rope", "B": B, "S": S, "HQ": HQ, "HK": HK, "D": D, "train": train, "norm": norm, "half": half,
            "dtype": dtype, "pos": pos, "each": each}
    return {"name": name, **case} if name else case


def _adapters(name, R, T, K, N, r, n, train=False, dtype="bf16", ragged=False):
    """R requests of T tokens together, adapters of rank r beside a K -> N projection, n of them; ``ragged``:
    requests of any lengths, some without an adapter, and tokens behind the last one."""
    case = {"kind": "adapters", "R": R, "T": T, "K": K, "N": N, "r": r, "n": n, "train": train, "dtype": dtype,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def _qkv(name, B, S, H, K, r, n, train=False):
    case = {"kind": "qkv", "B": B, "S": S, "H": H, "K": K, "r": r, "n": n, "train": train}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one token of each of four requests: latency
        _rope("rope_one", 4, 1, 30, 30, 128, each=True),
        # q and k of one of 8 ranks' tokens, in training
        _rope("rope_rank256", 1, 256, 30, 30, 128, train=True),
        # a video's sequence in training
        _rope("rope_long", 1, 8192, 30, 30, 128, train=True),
        # shared key heads, a width that is no power of two, fp32, positions between the whole numbers, two images
        _rope("rope_odd", 2, 1333, 14, 2, 72, half=True, dtype="fp32", pos="float32", each=True),
        # one token through the feed-forward's first Linear: latency
        _adapters("adapters_one", 1, 1, 3840, 10240, 16, 4),
        # the conditioning vectors of 32 requests through the modulation's Linear, an adapter each
        _adapters("adapters_cond", 32, 32, 256, 15360, 16, 32),
        # odd sizes, requests of any lengths, a 32-bit result
        _adapters("adapters_ragged", 13, 1333, 2570, 1001, 12, 5, dtype="fp32", ragged=True),
        # eight images through the feed-forward's first Linear
        _adapters("adapters_long", 8, 8192, 3840, 10240, 32, 8),
        # four adapters trained at once beside the attention's output projection
        _adapters("adapters_train", 4, 8192, 3840, 3840, 64, 4, train=True),
        # q, k, v of three small images with a style each
        _qkv("qkv_768", 3, 256, 30, 3840, 16, 3),
        # q, k, v of two large images
        _qkv("qkv_long", 2, 4096, 30, 3840, 16, 2),
        # the attention's adapters in training, one of 8 ranks' tokens
        _qkv("qkv_train768", 1, 768, 30, 3840, 16, 1, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Half the widths are multiples of 64, as models have them, half are any."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.5 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["rope", "rope", "adapters", "adapters", "adapters", "qkv"])
    if kind == "rope":
        B, S = rng.choice([1, 1, 2, 3]), _log_int(rng, 1, 16384)
        HQ, D = rng.randint(1, 32), rng.choice([128, 128, 8 * rng.randint(2, 32)])
        HK = rng.choice([HQ, HQ, rng.randint(1, HQ)])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        while B * S * (HQ + HK) * D * (2 if dtype == "bf16" else 4) > 8192 * 60 * 128 * 2:
            S = max(1, S // 2)
        return _rope(None, B, S, HQ, HK, D, rng.random() < 0.5, rng.random() < 0.8, rng.random() < 0.3, dtype,
                     rng.choice(["int32", "int64", "float32"]), rng.random() < 0.5)
    if kind == "adapters":
        T, K, N = _log_int(rng, 1, 16384), _width(rng, 64, 15360), _width(rng, 64, 15360)
        train, ragged, share = rng.random() < 0.4, rng.random() < 0.5, rng.random() < 0.3
        dtype = "bf16" if train else rng.choice(["bf16", "bf16", "fp32"])
        r = rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 128)])
        R = min(T, _log_int(rng, 1, 64))
        n = rng.randint(1, 32) if share else R
        while True:
            case = _adapters(None, R, T if ragged else T // R * R, K, N, r, n, train, dtype, ragged)
            w = work(case)
            if w["bytes"] <= 400e6 and w["flops"] <= 24e9 or T == R:
                return case
            T = max(R, T // 2)
    B, H = rng.randint(1, 4), rng.randint(1, 30)
    S = max(1, _log_int(rng, 1, 8192) // B)
    return _qkv(None, B, S, H, rng.choice([H * HEAD, H * HEAD, 64 * rng.randint(1, 60)]),
                rng.choice([8, 16, 16, 32, 64]), rng.choice([B, rng.randint(1, 8)]), rng.random() < 0.3 and B * S <= 2048)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int32": torch.int32, "int64": torch.int64,
          "float32": torch.float32}


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _activations(g, T, C):
    """Normal values with a few channels eight times as large, as hidden states have them."""
    x = torch.randn((T, C), device=DEV, generator=g)
    x *= 1.0 + 7.0 * (torch.rand(C, device=DEV, generator=g) < 0.01)
    return x.to(torch.bfloat16)


def _norm_weight(g, n):
    return (1.0 + _normal(g, n, scale=0.1, dtype=torch.float32)).to(torch.bfloat16)


def axes_of(D):
    """Widths of the (time, height, width) axes of a head of D features: a quarter and the rest in even halves."""
    t = D // 8 * 2
    h = (D - t) // 4 * 2
    return (t, h, D - t - h)


def _positions(g, B, S, kind, each):
    """A caption along the first axis, then an image's grid: [S, 3], or [B, S, 3] with another start for each."""
    i = torch.arange(S, device=DEV)
    text = S // 8
    wide = max(1, math.isqrt(max(1, S - text)))
    j = (i - text).clamp_min(0)
    image = i >= text
    p = torch.stack((torch.where(image, text, i), j // wide * image, j % wide * image), -1)
    if each:
        p = p + torch.randint(0, 1000, (B, 1, 3), device=DEV, generator=g)
    if kind == "float32":  # an image that was made larger: positions a fraction apart
        return p.float() * 0.37
    return p.to(_TYPES[kind])


def _low_rank(g, n, r, K, N):
    """A [n, r, K], B [n, N, r] and scales [n] of trained adapters: their result is about half the projection's."""
    a = _normal(g, n, r, K, scale=K ** -0.5)
    b = _normal(g, n, N, r, scale=0.5 * r ** -0.5)
    return a, b, torch.rand(n, device=DEV, generator=g) + 0.5


def _requests(g, R, T, n, ragged):
    """(adapter of each request, first token of each and the end, or None where all are T / R long)."""
    index = torch.randperm(max(n, R), device=DEV, generator=g)[:R] % n
    if not ragged:
        return index.int(), None
    index = torch.where(torch.rand(R, device=DEV, generator=g) < 0.2, -1, index)
    cuts = torch.randint(0, T - T // 16 + 1, (R + 1,), device=DEV, generator=g).sort().values
    cuts[0] = 0
    return index.int(), cuts.int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) + 3407)
    st = {"case": case}
    if case["kind"] == "rope":
        B, S, D, train = case["B"], case["S"], case["D"], case["train"]
        dt = _TYPES[case["dtype"]]
        for t, H in (("q", case["HQ"]), ("k", case["HK"])):
            st[t] = _normal(g, B, S, H, D, dtype=dt).transpose(1, 2).requires_grad_(train)
            st["w" + t] = _norm_weight(g, D).requires_grad_(train) if case["norm"] else None
            st["d" + t] = _normal(g, B, S, H, D, dtype=dt).transpose(1, 2) if train else None
        st["pos"] = _positions(g, B, S, case["pos"], case["each"])
        if own:
            import harp_amd

            st["rope"] = harp_amd.AxialRope(axes_of(D), THETA, layout="half" if case["half"] else "interleaved")
        return st
    if case["kind"] == "adapters":
        T, K, N, train = case["T"], case["K"], case["N"], case["train"]
        st["x"] = _activations(g, T, K).requires_grad_(train)
        st["y"] = _normal(g, T, N, dtype=_TYPES[case["dtype"]])
        st["a"], st["b"], st["s"] = _low_rank(g, case["n"], case["r"], K, N)
        st["index"], st["offsets"] = _requests(g, case["R"], T, case["n"], case["ragged"])
        if train:
            st["dy"] = _normal(g, T, N)
            st["a"].requires_grad_(), st["b"].requires_grad_()
        if own:
            import harp_amd

            st["adapters"] = harp_amd.Adapters(st["a"], st["b"], st["s"])
            st["requests"] = harp_amd.AdapterRequests(st["index"], st["offsets"])
        return st
    B, S, H, K, train = case["B"], case["S"], case["H"], case["K"], case["train"]
    N = H * HEAD
    st["x"] = _activations(g, B * S, K).view(B, S, K).requires_grad_(train)
    st["w"] = [_normal(g, N, K, scale=K ** -0.5) for _ in range(3)]
    st["low"] = [_low_rank(g, case["n"], case["r"], K, N) for _ in range(3)]
    st["nw"] = [_norm_weight(g, HEAD) for _ in range(2)]
    st["index"], _ = _requests(g, B, B * S, case["n"], False)
    st["pos"] = _positions(g, B, S, "int32", True)
    if train:
        st["d"] = [_normal(g, B, S, H, HEAD).transpose(1, 2) for _ in range(3)]
        for a, b, _ in st["low"]:
            a.requires_grad_(), b.requires_grad_()
    if own:
        import harp_amd

        to = [SimpleNamespace(weight=w, bias=None) for w in st["w"]]
        norms = [SimpleNamespace(weight=nw, eps=EPS) for nw in st["nw"]]
        attn = SimpleNamespace(heads=H, to_q=to[0], to_k=to[1], to_v=to[2], norm_q=norms[0], norm_k=norms[1])
        low = [harp_amd.Adapters(*abs_) for abs_ in st["low"]]
        st["attn"] = harp_amd.adapt_attention(attn, to_q=low[0], to_k=low[1], to_v=low[2])
        st["requests"] = harp_amd.AdapterRequests(st["index"])
        st["positions"] = harp_amd.AxialPositions(st["pos"], harp_amd.AxialRope(axes_of(HEAD), THETA))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    import harp_amd

    case = st["case"]
    if case["kind"] == "rope":
        out = harp_amd.qk_norm_axial_rope(st["q"], st["k"], st["pos"], st["rope"], st["wq"], st["wk"],
                                          EPS if case["norm"] else None)
        if not case["train"]:
            return out
        wrt = (st["q"], st["k"]) + ((st["wq"], st["wk"]) if case["norm"] else ())
        return (*out, *torch.autograd.grad(out, wrt, (st["dq"], st["dk"])))
    if case["kind"] == "adapters":
        out = harp_amd.add_adapters(st["y"], st["x"], st["adapters"], st["requests"])
        if not case["train"]:
            return out
        return (out, *torch.autograd.grad(out, (st["x"], st["a"], st["b"]), st["dy"]))
    attn = st["attn"]
    out = harp_amd.project_qkv(attn, st["x"], st["positions"], requests=st["requests"])
    if not case["train"]:
        return out
    wrt = (st["x"], attn.to_q.a, attn.to_q.b, attn.to_k.a, attn.to_k.b, attn.to_v.a, attn.to_v.b)
    return (*out, *torch.autograd.grad(out, wrt, st["d"]))


def _cos_sin(pos, D):
    """cos and sin of every pair's angle, [B or 1, 1, S, D/2] in 32 bits, from angles in 64."""
    axes = axes_of(D)
    inv = torch.cat([THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d) for d in axes])
    axis = torch.repeat_interleave(torch.arange(len(axes), device=DEV), torch.tensor(axes, device=DEV) // 2,
                                   output_size=D // 2)
    ang = pos.double()[..., axis] * inv
    ang = ang.unsqueeze(-3) if ang.dim() == 3 else ang[None, None]
    return torch.cos(ang).float(), torch.sin(ang).float()


def _rotate(x, cos, sin, half):
    if half:
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _rms(x):
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _norm_rope_plain(x, w, cos, sin, half):
    if w is not None:
        x = x * _rms(x) * w.float()
    return _rotate(x, cos, sin, half)


def _norm_rope_back_plain(d, x, w, cos, sin, half):
    """(gradient of x, of w) in 32 bits."""
    d = _rotate(d, cos, -sin, half)
    if w is None:
        return d, None
    r = _rms(x)
    n = x * r
    gw = (d * n).sum((0, 1, 2))
    d = d * w.float()
    return r * (d - n * (d * n).mean(-1, keepdim=True)), gw


def _mine(index, offsets, T, n):
    """[T, n, 1]: whether token t takes adapter i."""
    t = torch.arange(T, device=DEV)
    if offsets is None:
        who = index.long().repeat_interleave(T // index.numel())
    else:
        request = torch.searchsorted(offsets[1:].contiguous(), t, right=True)
        inside = request < index.numel()
        who = torch.where(inside, index.long()[request.clamp_max(index.numel() - 1)], -1)
    return (who[:, None] == torch.arange(n, device=DEV))[..., None]


def _low_plain(x, mine, a, s):
    """s x A^T of each token's adapter, zeros in the others' places: [T, n r]."""
    n, r, K = a.shape
    t = (x @ a.float().reshape(n * r, K).t()).view(-1, n, r) * s[:, None]
    return torch.where(mine, t, 0.0).flatten(1)


def _stacked(b):
    """B of all adapters side by side: [N, n r]."""
    return b.float().permute(1, 0, 2).flatten(1)


def _low_back_plain(d, t, x, mine, a, b, s):
    """Gradients (x, a, b) of t = _low_plain(x) through d = gradient of t B^T."""
    n, r, K = a.shape
    u = torch.where(mine, (d @ _stacked(b)).view(-1, n, r) * s[:, None], 0.0).flatten(1)
    gb = (d.t() @ t).view(-1, n, r).permute(1, 0, 2)
    return u @ a.float().reshape(n * r, K), (u.t() @ x).view(n, r, K).to(a.dtype), gb.to(b.dtype)


def _run_plain(st):
    case = st["case"]
    if case["kind"] == "rope":
        half, dt = case["half"], st["q"].dtype
        cos, sin = _cos_sin(st["pos"], case["D"])
        q, k = st["q"].detach().float(), st["k"].detach().float()
        wq, wk = st["wq"], st["wk"]
        if case["norm"]:
            wq, wk = wq.detach(), wk.detach()
        out = (_norm_rope_plain(q, wq, cos, sin, half).to(dt), _norm_rope_plain(k, wk, cos, sin, half).to(dt))
        if not case["train"]:
            return out
        gq, gwq = _norm_rope_back_plain(st["dq"].float(), q, wq, cos, sin, half)
        gk, gwk = _norm_rope_back_plain(st["dk"].float(), k, wk, cos, sin, half)
        out += (gq.to(dt), gk.to(dt))
        return out + ((gwq.to(wq.dtype), gwk.to(wk.dtype)) if case["norm"] else ())
    if case["kind"] == "adapters":
        x, a, b, s = st["x"].detach().float(), st["a"].detach(), st["b"].detach(), st["s"]
        mine = _mine(st["index"], st["offsets"], case["T"], case["n"])
        t = _low_plain(x, mine, a, s)
        out = (st["y"].float() + t @ _stacked(b).t()).to(st["y"].dtype)
        if not case["train"]:
            return out
        gx, ga, gb = _low_back_plain(st["dy"].float(), t, x, mine, a, b, s)
        return out, gx.to(st["x"].dtype), ga, gb
    B, S, H = case["B"], case["S"], case["H"]
    x = st["x"].detach().float().flatten(0, 1)
    cos, sin = _cos_sin(st["pos"], HEAD)
    mine = _mine(st["index"], None, B * S, case["n"])
    nw = (*st["nw"], None)
    w = [w.float() for w in st["w"]]
    low = [(a.detach(), b.detach(), s) for a, b, s in st["low"]]
    t = [_low_plain(x, mine, a, s) for a, _, s in low]
    y = [x @ w[i].t() + t[i] @ _stacked(low[i][1]).t() for i in (0, 1, 2)]
    y = [v.view(B, S, H, HEAD).transpose(1, 2) for v in y]
    out = tuple((_norm_rope_plain(v, n, cos, sin, False) if n is not None else v).to(torch.bfloat16)
                for v, n in zip(y, nw))
    if not case["train"]:
        return out
    d = [v.float() for v in st["d"]]
    d = [_norm_rope_back_plain(d[i], y[i], nw[i], cos, sin, False)[0] if nw[i] is not None else d[i] for i in (0, 1, 2)]
    d = [v.transpose(1, 2).reshape(B * S, -1) for v in d]
    back = [_low_back_plain(d[i], t[i], x, mine, *low[i]) for i in (0, 1, 2)]
    gx = d[0] @ w[0] + d[1] @ w[1] + d[2] @ w[2] + back[0][0] + back[1][0] + back[2][0]
    return (*out, gx.to(torch.bfloat16).view(B, S, -1), *(gr for _, ga, gb in back for gr in (ga, gb)))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

_BYTES = {"bf16": 2, "fp32": 4, "int32": 4, "int64": 8, "float32": 4}


def work(case):
    if case["kind"] == "rope":
        n = case["B"] * case["S"] * (case["HQ"] + case["HK"]) * case["D"]
        pos = 3 * case["S"] * (case["B"] if case["each"] else 1) * _BYTES[case["pos"]]
        # in and out; in training the outputs' gradients in and the inputs' out as well
        return {"bytes": (4 if case["train"] else 2) * n * _BYTES[case["dtype"]] + pos,
                "flops": ((8 if case["norm"] else 3) + (14 if case["norm"] else 3) * case["train"]) * n}
    T = case["T"] if case["kind"] == "adapters" else case["B"] * case["S"]
    used = min(case["n"], case["R"] if case["kind"] == "adapters" else case["B"])
    K, r, train = case["K"], case["r"], case["train"]
    if case["kind"] == "adapters":
        N = case["N"]
        low = used * r * (K + N) * 2 + (case["n"] * r * (K + N) * 2 if train else 0)
        # x and the projection's result in, the sum out; in training dy in, dx out
        return {"bytes": T * K * 2 + 2 * T * N * _BYTES[case["dtype"]] + low + (T * (K + N) * 2 if train else 0),
                "flops": (6 if train else 2) * T * r * (K + N)}
    N = 3 * case["H"] * HEAD
    low = (used + case["n"] * train) * r * (3 * K + N) * 2
    # x and the weights in, q, k, v out; in training their gradients in and x's out
    return {"bytes": (2 if train else 1) * T * (K + N) * 2 + N * K * 2 + low,
            "flops": (4 if train else 2) * T * N * K + (6 if train else 2) * T * r * (3 * K + N)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _turned(x, pos, half):
    """Complex multiplication of the pairs of x [B, H, S, D] by exp(i angle)."""
    D = x.shape[-1]
    phase, first = [], 0
    for a, d in enumerate(axes_of(D)):
        rates = torch.tensor([THETA ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device=DEV)
        phase.append(pos[..., a, None].double() * rates)
    ang = torch.cat(phase, -1)
    if ang.dim() == 3:
        ang = ang.unsqueeze(1)
    turn = torch.polar(torch.ones_like(ang), ang)
    if half:
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)
    return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (D // 2, 2)).contiguous()) * turn).flatten(-2)


def _normed64(x, w):
    return x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w


def _delta64(x, a, b, s, index, offsets):
    """The adapters' part, one request after the other: [T, N]."""
    T = x.shape[0]
    ends = [i * (T // len(index)) for i in range(len(index) + 1)] if offsets is None else offsets.tolist()
    parts = [x.new_zeros(ends[0], b.shape[1])]
    for i, which in enumerate(index.tolist()):
        rows = x[ends[i]:ends[i + 1]]
        parts.append(rows.new_zeros(len(rows), b.shape[1]) if which < 0
                     else s[which].double() * ((rows @ a[which].t()) @ b[which].t()))
    parts.append(x.new_zeros(T - ends[-1], b.shape[1]))
    return torch.cat(parts)


def exact(case, seed):
    st = prepare(case, seed)
    train = case["train"]

    def leaf(t):
        return t.detach().double().requires_grad_(train)

    with torch.set_grad_enabled(train):
        if case["kind"] == "rope":
            leaves, out, weights = [], [], []
            for t in ("q", "k"):
                x = y = leaf(st[t])
                leaves.append(x)
                if case["norm"]:
                    weights.append(leaf(st["w" + t]))
                    y = _normed64(x, weights[-1])
                out.append(_turned(y, st["pos"], case["half"]))
            leaves, down = leaves + weights, [st["dq"], st["dk"]]
        elif case["kind"] == "adapters":
            leaves = [leaf(st[t]) for t in ("x", "a", "b")]
            out = [st["y"].double() + _delta64(*leaves, st["s"], st["index"], st["offsets"])]
            down = [st.get("dy")]
            if not train:
                return out[0]
        else:
            x = leaf(st["x"])
            leaves, out, down = [x], [], st.get("d")
            flat = x.flatten(0, 1)
            for i, (a, b, s) in enumerate(st["low"]):
                a, b = leaf(a), leaf(b)
                leaves += [a, b]
                y = flat @ st["w"][i].double().t() + _delta64(flat, a, b, s, st["index"], None)
                y = y.view(case["B"], case["S"], case["H"], HEAD).permute(0, 2, 1, 3)
                out.append(y if i == 2 else _turned(_normed64(y, st["nw"][i].double()), st["pos"], False))
        if train:
            grads = torch.autograd.grad(out, leaves, [d.double() for d in down])
    out = tuple(t.detach() for t in out)
    return out + tuple(grads) if train else out
