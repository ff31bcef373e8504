"""Performance cases of the operators around the attention block: the residual
addition with its RMSNorm, and the block's Linear layers in 8-bit integers.

Every case is a plain dict; ``prepare`` makes what a user's program holds
before the call (inputs, quantised weights, modules), ``run`` is one pass,
``exact`` is the same result in 64 bits.  Kinds:

* ``norm``: :func:`harp_amd.add_rms_norm` in training, forward + backward;
* ``norm8``: :func:`harp_amd.add_rms_norm_int8` (``norm`` true) or
  :func:`harp_amd.quantize_int8`, 8-bit rows with a scale for each;
* ``linear``: :class:`harp_amd.Int8Linear`, on bf16 activations or on 8-bit
  rows (``rows``);
* ``qkv``: :func:`harp_amd.project_qkv` on an attention module with
  :class:`harp_amd.Int8Linear` projections.

With ``own`` false ``run`` computes the operators from elementary torch
operations in 32 bits instead.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
HEAD = 128


def _norm(name, T, C, res="bf16", w="bf16", pad=0):
    """T tokens of C channels, the last ``pad`` of them padding (zeros); residual and weight types."""
    case = {"kind": "norm", "T": T, "C": C, "res": res, "w": w, "pad": pad}
    return {"name": name, **case} if name else case


def _norm8(name, T, C, norm=True, res="bf16", w="bf16", pad=0):
    case = {"kind": "norm8", "T": T, "C": C, "norm": norm, "res": res, "w": w, "pad": pad}
    return {"name": name, **case} if name else case


def _linear(name, T, N, K, rows=False, bias="none", out="bf16"):
    case = {"kind": "linear", "T": T, "N": N, "K": K, "rows": rows, "bias": bias, "out": out}
    return {"name": name, **case} if name else case


def _qkv(name, B, S, H, K, rows=True, w="bf16"):
    case = {"kind": "qkv", "B": B, "S": S, "H": H, "K": K, "rows": rows, "w": w}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the norm before attention or the feed-forward in training, the tokens of one of 8 ranks
        _norm("norm_rank256", 256, 3840),
        # a width that no vector load divides, with an fp32 weight and padding at the end
        _norm("norm_odd", 1333, 2561, w="fp32", pad=29),
        # a long sequence with the residual stream in 32 bits
        _norm("norm_long", 8192, 3840, res="fp32"),
        # one token through the norm in front of an 8-bit layer: latency
        _norm8("norm8_one", 1, 3840),
        # a long sequence through it
        _norm8("norm8_long", 8192, 3840),
        # one conditioning vector through a feed-forward Linear: the weights' bytes
        _linear("linear_one", 1, 10240, 3840),
        # a handful of tokens through the feed-forward's second Linear
        _linear("linear_few", 19, 3840, 10240, rows=True, bias="bf16"),
        # the feed-forward's first Linear at one rank's tokens
        _linear("linear_rank768", 768, 10240, 3840, rows=True),
        # odd sizes, a bias and a 32-bit result
        _linear("linear_ragged", 1333, 1001, 2570, bias="fp32", out="fp32"),
        # the feed-forward's first Linear over a long sequence
        _linear("linear_long", 8192, 10240, 3840, rows=True),
        # q, k, v of a small image's tokens
        _qkv("qkv_256", 1, 256, 30, 3840),
        # q, k, v of a long sequence
        _qkv("qkv_long", 1, 8192, 30, 3840),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Half the widths are multiples of 64, as models have them, half are any."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.5 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm8", "norm8", "linear", "linear", "linear", "qkv", "qkv"])
    w = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("norm", "norm8"):
        T, C = _log_int(rng, 1, 16384), _width(rng, 64, 10240)
        while T * C > 8192 * 3840:
            T = max(1, T // 2)
        res, pad = rng.choice(["bf16", "bf16", "fp32"]), rng.choice([0, 0, rng.randint(0, T // 8)])
        if kind == "norm":
            return _norm(None, T, C, rng.choice([res, "none"]), w, pad)
        return _norm8(None, T, C, rng.random() < 0.7, rng.choice([res, "none"]), w, pad)
    if kind == "linear":
        while True:
            T, N, K = _log_int(rng, 1, 8192), _width(rng, 64, 15360), _width(rng, 64, 15360)
            if T * N * K <= 8192 * 10240 * 3840:
                return _linear(None, T, N, K, rng.random() < 0.5, rng.choice(["none", "bf16", "fp32"]),
                               rng.choice(["bf16", "bf16", "fp32"]))
    B, S, H = rng.choice([1, 1, 2]), _log_int(rng, 1, 8192), rng.randint(1, 30)
    while B * S > 8192:
        S //= 2
    return _qkv(None, B, S, H, rng.choice([H * HEAD, H * HEAD, 16 * rng.randint(4, 240)]), rng.random() < 0.5, w)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _activations(g, T, C, dtype=torch.bfloat16, pad=0):
    """Normal values with a few channels eight times as large, as hidden states have them."""
    x = torch.randn((T, C), device=DEV, generator=g)
    x *= 1.0 + 7.0 * (torch.rand(C, device=DEV, generator=g) < 0.01)
    x[T - pad:] = 0.0
    return x.to(dtype)


def _quantise(y):
    """(values in -127 .. 127 as floats, scale of each row): y is about values * scale.

    The quotient is formed in 64 bits: in 32, one value in a million lands on
    the other side of the border between two steps."""
    amax = y.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * y.double() / amax.double()).float()
    return torch.where(amax > 0, q, torch.zeros_like(q)), amax / 127.0


def _int8_rows(y):
    """8-bit rows of y and their scales, the storage's rows padded to 16 bytes."""
    q, s = _quantise(y.float())
    T, C = q.shape
    store = torch.zeros((T, (C + 15) // 16 * 16), dtype=torch.int8, device=DEV)
    store[:, :C] = q.to(torch.int8)
    return store[:, :C], s.squeeze(-1).contiguous()


def _norm_weight(g, n, kind):
    return (1.0 + _normal(g, n, scale=0.1, dtype=torch.float32)).to(_TYPES[kind])


def _freqs(S):
    """The RoPE table: exp(i * position * theta^(-2p/D)), complex64 [S, D/2]."""
    inv = 256.0 ** (-torch.arange(0, HEAD, 2, dtype=torch.float64) / HEAD)
    ang = torch.arange(S, dtype=torch.float64)[:, None] * inv[None, :]
    return torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) + 3407)
    st = {"case": case}
    if case["kind"] in ("norm", "norm8"):
        T, C, train = case["T"], case["C"], case["kind"] == "norm"
        st["x"] = _activations(g, T, C, pad=case["pad"]).requires_grad_(train)
        st["w"] = _norm_weight(g, C, case["w"]).requires_grad_(train)
        st["res"] = None
        if case["res"] != "none":
            st["res"] = _activations(g, T, C, _TYPES[case["res"]], case["pad"]).requires_grad_(train)
        if train:
            st["dy"] = _normal(g, T, C)
            st["dh"] = _normal(g, T, C, dtype=st["res"].dtype) if st["res"] is not None else None
        return st
    if case["kind"] == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        x = _activations(g, T, K)
        st["x"] = _int8_rows(x) if case["rows"] else x
        st["wq"], st["ws"] = _int8_rows(_normal(g, N, K, scale=K ** -0.5, dtype=torch.float32))
        st["bias"] = None if case["bias"] == "none" else _normal(g, N, scale=0.1, dtype=_TYPES[case["bias"]])
        if own:
            import harp_amd

            st["layer"] = harp_amd.Int8Linear.from_quantized(st["wq"], st["ws"], st["bias"],
                                                             out_dtype=_TYPES[case["out"]])
            if case["rows"]:
                st["rows"] = harp_amd.Int8Rows(*st["x"])
        return st
    B, S, H, K = case["B"], case["S"], case["H"], case["K"]
    x = _activations(g, B * S, K)
    st["x"] = _int8_rows(x) if case["rows"] else x.view(B, S, K)
    st["proj"] = [_int8_rows(_normal(g, H * HEAD, K, scale=K ** -0.5, dtype=torch.float32)) for _ in range(3)]
    st["nw"] = [_norm_weight(g, HEAD, case["w"]) for _ in range(2)]
    st["freqs"] = _freqs(S)
    if own:
        import harp_amd

        to = [harp_amd.Int8Linear.from_quantized(wq, ws) for wq, ws in st["proj"]]
        norms = [SimpleNamespace(weight=nw, eps=EPS) for nw in st["nw"]]
        st["attn"] = SimpleNamespace(heads=H, to_q=to[0], to_k=to[1], to_v=to[2], norm_q=norms[0], norm_k=norms[1])
        if case["rows"]:
            q, s = st["x"]
            st["rows"] = harp_amd.Int8Rows(q.unflatten(0, (B, S)), s.view(B, S))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    import harp_amd

    case = st["case"]
    if case["kind"] == "norm":
        y, h = harp_amd.add_rms_norm(st["x"], st["res"], st["w"], EPS)
        if st["res"] is None:
            return (y, *torch.autograd.grad(y, (st["x"], st["w"]), st["dy"]))
        return (y, h, *torch.autograd.grad((y, h), (st["x"], st["res"], st["w"]), (st["dy"], st["dh"])))
    if case["kind"] == "norm8":
        if not case["norm"]:
            rows = harp_amd.quantize_int8(st["x"])
            return rows.dequantize(), rows.scales
        rows, h = harp_amd.add_rms_norm_int8(st["x"], st["res"], st["w"], EPS)
        return (rows.dequantize(), rows.scales) + ((h,) if st["res"] is not None else ())
    x = st["rows"] if case["rows"] else st["x"]
    if case["kind"] == "linear":
        return st["layer"](x)
    return harp_amd.project_qkv(st["attn"], x, st["freqs"])


def _rms_plain(h):
    return torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)


def _run_plain(st):
    case = st["case"]
    if case["kind"] == "norm":
        return _norm_plain(st["x"].detach(), None if st["res"] is None else st["res"].detach(), st["w"].detach(),
                           st["dy"], st["dh"])
    if case["kind"] == "norm8":
        x, res, h = st["x"], st["res"], None
        y = x.float()
        if case["norm"]:
            if res is not None:
                h = (y + res.float()).to(res.dtype)
                y = h.float()
            y = y * _rms_plain(y) * st["w"].float()
        q, s = _quantise(y)
        out = ((q * s).to(torch.bfloat16), s.squeeze(-1))
        return out + ((h,) if h is not None else ())
    q, s = (st["x"][0].float(), st["x"][1][:, None]) if case["rows"] else _quantise(st["x"].float())
    if case["kind"] == "linear":
        y = (q @ st["wq"].float().t()) * s * st["ws"]
        if st["bias"] is not None:
            y = y + st["bias"].float()
        return y.to(_TYPES[case["out"]])
    B, S, H = case["B"], case["S"], case["H"]
    q, s = q.reshape(B, S, -1), s.reshape(B, S, 1)
    cos, sin = st["freqs"].real, st["freqs"].imag
    outs = []
    for i, (wq, ws) in enumerate(st["proj"]):
        y = ((q @ wq.float().t()) * s * ws).unflatten(-1, (H, HEAD)).transpose(1, 2)
        if i < 2:
            y = y * _rms_plain(y) * st["nw"][i].float()
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        outs.append(y.to(torch.bfloat16))
    return tuple(outs)


def _norm_plain(x, res, w, dy, dh):
    h = x if res is None else (x.float() + res.float()).to(res.dtype)
    hf, wf, d = h.float(), w.float(), dy.float()
    r = _rms_plain(hf)
    n = hf * r
    y = (n * wf).to(x.dtype)
    gw = (d * n).sum(0).to(w.dtype)
    d = d * wf
    dx = r * (d - n * (d * n).mean(-1, keepdim=True))
    if res is None:
        return y, dx.to(x.dtype), gw
    dx = dx + dh.float()
    return y, h, dx.to(x.dtype), dx.to(res.dtype), gw


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

_BYTES = {"none": 0, "bf16": 2, "fp32": 4}


def work(case):
    if case["kind"] in ("norm", "norm8"):
        n, res = case["T"] * case["C"], _BYTES[case["res"]]
        if case["kind"] == "norm":
            # x, residual, dy, dh in; y, h and the gradient(s) of x and the residual out
            per = 2 + 2 + 2 + 2 + 3 * res - (2 if res == 2 else 0)
            return {"bytes": n * per + 2 * case["C"] * _BYTES[case["w"]], "flops": 18 * n}
        # x, residual in; h, the 8-bit values and their scales out
        per = 2 + 1 + (2 * res if case["norm"] else 0)
        return {"bytes": n * per + 4 * case["T"], "flops": (8 if case["norm"] else 3) * n}
    if case["kind"] == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        x = T * K + 4 * T if case["rows"] else 2 * T * K
        return {"bytes": x + N * K + 4 * N + _BYTES[case["bias"]] * N + _BYTES[case["out"]] * T * N,
                "flops": 2 * T * N * K}
    T, N, K = case["B"] * case["S"], 3 * case["H"] * HEAD, case["K"]
    x = T * K + 4 * T if case["rows"] else 2 * T * K
    return {"bytes": x + N * K + 4 * N + 2 * T * N + 4 * HEAD * case["S"], "flops": 2 * T * N * K}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _rows64(x):
    """The 8-bit values and scales of x's rows, by their definition: the nearest of -127 .. 127 steps of max / 127.

    127 x is exact before the division: half the maximum lies halfway between
    two steps, and goes to the even one."""
    most = x.abs().max(dim=-1, keepdim=True).values
    return torch.round(torch.where(most == 0, torch.zeros_like(x), 127 * x / most)), most / 127


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        x, w = (st[k].detach().double().requires_grad_(True) for k in ("x", "w"))
        # the addition's result is kept, and normalised, in the residual's type
        h = x
        if st["res"] is not None:
            h = (x + st["res"].double()).to(st["res"].dtype).detach().double().requires_grad_(True)
        y = h / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + EPS) * w
        if st["res"] is None:
            return (y.detach(), *torch.autograd.grad(y, (x, w), st["dy"].double()))
        gh, gw = torch.autograd.grad(y, (h, w), st["dy"].double())
        gh = gh + st["dh"].double()
        return y.detach(), h.detach(), gh, gh, gw
    if case["kind"] == "norm8":
        y, h = st["x"].double(), None
        if case["norm"]:
            if st["res"] is not None:
                h = y = (y + st["res"].double()).to(st["res"].dtype).double()
            y = y / torch.sqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * st["w"].double()
        steps, step = _rows64(y)
        return (steps * step, step[:, 0]) + (() if h is None else (h,))
    if case["rows"]:
        x = st["x"][0].double() * st["x"][1].double().unsqueeze(1)
    else:
        steps, step = _rows64(st["x"].double())
        x = steps * step
    if case["kind"] == "linear":
        y = x @ (st["wq"].double() * st["ws"].double().unsqueeze(1)).t()
        return y if st["bias"] is None else y + st["bias"].double()
    x = x.reshape(case["B"] * case["S"], -1)
    res = []
    for i, (wq, ws) in enumerate(st["proj"]):
        y = (x @ (wq.double() * ws.double().unsqueeze(1)).t()).view(case["B"], case["S"], case["H"], HEAD)
        y = y.permute(0, 2, 1, 3)
        if i < 2:
            y = y / torch.sqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * st["nw"][i].double()
            turned = torch.view_as_complex(y.unflatten(-1, (HEAD // 2, 2)).contiguous()) * st["freqs"].to(torch.complex128)
            y = torch.view_as_real(turned).flatten(-2)
        res.append(y)
    return tuple(res)
