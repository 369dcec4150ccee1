"""Timing cases of the operators of a quantized feed-forward block, through rt4_amd's public functions.

Five operators, at the 27B layer shapes (hidden size 5120, feed-forward size 17408) and sizes around them:

* ``linear``: ``gemm_w8a8``, the product of int8 activations (a scale for each token) and int8 weights (a scale for each
  channel), for layers that are kept at 8 bits.
* ``gated``:  ``ffn_gate_w8a8``, the first half of a gated feed-forward block on such weights: both products, the
  activation and the product of the two.
* ``gated4``: ``ffn_gate_w4a8``, the same on RT4 weights for the 1-4 rows of a decode step.
* ``norm``:   ``block_norm``, what stands between one block and the next: the block's output normed, gated and scaled, added
  to the residual, the residual normed for the next block and quantized in the form that its products read.
* ``quant``:  ``quant_token_a8``, activations to int8 with a scale for each token.

Codes are the library's public format and every code has one right value (the nearest integer to 127 x / max|x|, decided in
64 bits), so they are compared as the whole numbers that they are, beside the scales that give them their values.
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

DEV = "cuda"
G = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One token through a square projection: latency and the read of 26 MB of weights.
        {"name": "linear_m1", "kind": "linear", "M": 1, "N": 5120, "K": 5120, "out": "f32"},
        # A small ragged batch and a layer whose sizes divide by nothing.
        {"name": "linear_m37_odd", "kind": "linear", "M": 37, "N": 4999, "K": 7056, "out": "bf16"},
        # A prompt of 1024 tokens through the down projection.
        {"name": "linear_m1024_down", "kind": "linear", "M": 1024, "N": 5120, "K": 17408, "out": "bf16"},
        # A long prompt through the up projection: the largest product.
        {"name": "linear_m4096_up", "kind": "linear", "M": 4096, "N": 17408, "K": 5120, "out": "bf16"},
        # One token through the first half of the feed-forward block: 178 MB of weights.
        {"name": "gated_m1", "kind": "gated", "M": 1, "N": 17408, "K": 5120, "act": "silu", "out": "f32"},
        # A prompt of an odd length through the same.
        {"name": "gated_m1000", "kind": "gated", "M": 1000, "N": 17408, "K": 5120, "act": "silu", "out": "bf16"},
        # The verify step of a token and three drafts, RT4 weights.
        {"name": "gated4_m4", "kind": "gated4", "M": 4, "N": 17408, "K": 5120, "act": "silu"},
        # One token through a small RT4 layer of odd width.
        {"name": "gated4_m1_small", "kind": "gated4", "M": 1, "N": 2051, "K": 2048, "act": "gelu_tanh"},
        # Between two blocks of a decode step: the residual is f32, the next products are RT4 decode linears.
        {"name": "norm_m4_act", "kind": "norm", "M": 4, "K": 5120, "y": "f32", "h": "f32", "post": False, "gate": "none", "n": "act"},
        # Between two blocks of a long prompt, with a norm behind the block and a gate for each channel; token codes.
        {"name": "norm_m4096_token", "kind": "norm", "M": 4096, "K": 5120, "y": "bf16", "h": "bf16", "post": True, "gate": "channel", "n": "token"},
        # Four tokens between the two halves of the feed-forward block.
        {"name": "quant_m4", "kind": "quant", "M": 4, "K": 17408, "x": "f32"},
        # A prompt of an odd length between them.
        {"name": "quant_m1000", "kind": "quant", "M": 1000, "K": 17408, "x": "bf16"},
    ]


MOST = 4096 * 17408 * 5120


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "gated", "gated", "gated4", "norm", "norm", "quant"])
    out = rng.choice(["f32", "bf16", "f16"])
    if kind in ("linear", "gated"):
        M, N, K = _log(rng, 1, 4096), _log(rng, 16, 20000), 16 * _log(rng, 4, 1100)
        while M * N * K * (2 if kind == "gated" else 1) > MOST:
            M = (M + 1) // 2
        c = {"kind": kind, "M": M, "N": N, "K": K, "out": out}
        return c | {"act": rng.choice(["silu", "gelu_tanh"])} if kind == "gated" else c
    if kind == "gated4":
        return {"kind": kind, "M": rng.randint(1, 4), "N": _log(rng, 100, 17408), "K": 128 * _log(rng, 4, 136), "act": rng.choice(["silu", "gelu_tanh"])}
    if kind == "quant":
        return {"kind": kind, "M": _log(rng, 1, 4096), "K": _log(rng, 64, 17408), "x": out}
    n = rng.choice(["f32", "bf16", "token", "act", "rows"])
    K = 128 * _log(rng, 1, 136) if n in ("act", "rows") else _log(rng, 64, 17408)
    M = _log(rng, 1, 4096)
    while M * K > 4096 * 5120:
        M = (M + 1) // 2
    return {"kind": kind, "M": M, "K": K, "y": rng.choice(["none", "f32", "bf16"]), "h": rng.choice(["f32", "bf16", "f16"]),
            "post": rng.random() < 0.4, "gate": rng.choice(["none", "none", "channel", "token"]), "n": n}


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1 + seed)
    return g


def _codes8(rows, K, g, size):
    """int8 codes and scales of N(0, size^2) rows of K values, the rows a little unlike each other."""
    x = torch.randn((rows, K), device=DEV, generator=g)
    a = x.abs().amax(-1)
    q = x.mul_((127 / a)[:, None]).round_().to(torch.int8)
    return q, a * (size / 127) * (0.5 + torch.rand((rows,), device=DEV, generator=g))


def _rt4(N, K, g):
    """RT4 weights: codes uniform in [-8, 7], fp16 scales |N(0,1)| * 0.01 + 1e-3 (as bit patterns)."""
    wq = torch.randint(-2**31, 2**31, (N, K // 8), dtype=torch.int32, device=DEV, generator=g)
    ws = torch.randn((N, K // G), device=DEV, generator=g).abs() * 0.01 + 1e-3
    return wq, ws.to(torch.float16).view(torch.int16)


def prepare(case, seed):
    g = _gen(seed)
    kind, M, K = case["kind"], case["M"], case["K"]
    st = {"case": case}
    if kind in ("linear", "gated"):
        N = case["N"]
        st["x"], st["sx"] = _codes8(M, K, g, 1.0)
        st["w"], st["sw"] = _codes8(N, K, g, K ** -0.5)
        if kind == "gated":
            st["wu"], st["su"] = _codes8(N, K, g, K ** -0.5)
    elif kind == "gated4":
        N = case["N"]
        x = torch.randn((M, K // G, G), device=DEV, generator=g)
        s = x.abs().amax(-1, keepdim=True) / 127
        q = (x / s).round_().to(torch.int8).reshape(M, K // 8, 4, 2)
        st["x"], st["sx"] = q.transpose(-1, -2).reshape(M, K).contiguous(), s[..., 0].contiguous()    # even elements of 8, then odd ones
        st["w"], st["sw"] = _rt4(N, K, g)
        st["wu"], st["su"] = _rt4(N, K, g)
    elif kind == "norm":
        # A residual stream has a few channels far larger than the rest.
        loud = 1 + 30 * (torch.rand((K,), device=DEV, generator=g) < 0.004).float()
        st["h"] = (3 * torch.randn((M, K), device=DEV, generator=g) * loud).to(TYPES[case["h"]])
        st["weight"] = 1 + 0.2 * torch.randn((K,), device=DEV, generator=g)
        st["y"] = st["post_weight"] = st["gate"] = None
        if case["y"] != "none":
            st["y"] = torch.randn((M, K), device=DEV, generator=g).to(TYPES[case["y"]])
            if case["post"]:
                st["post_weight"] = 1 + 0.2 * torch.randn((K,), device=DEV, generator=g)
            if case["gate"] != "none":
                st["gate"] = torch.rand((K,) if case["gate"] == "channel" else (M, K), device=DEV, generator=g).to(TYPES[case["y"]])
    else:
        st["x"] = (torch.randn((M, K), device=DEV, generator=g) * torch.randn((M, K), device=DEV, generator=g)).to(TYPES[case["x"]])
    return st


# ------------------------------------------------------------------ passes --
SCALE, EPS = 0.7, 1e-6


def run(state):
    if own:
        return _run_own(state)
    return {"linear": _plain_linear, "gated": _plain_gated, "gated4": _plain_gated4, "norm": _plain_norm, "quant": _plain_quant}[state["case"]["kind"]](state)


_pkg = str(pathlib.Path(__file__).resolve().parents[1] / "k100lc-rt4_amd")


def _run_own(st):
    if "rt4_amd" not in sys.modules and _pkg not in sys.path:
        sys.path.insert(0, _pkg)
    import rt4_amd
    c = st["case"]
    if c["kind"] == "linear":
        return {"out": rt4_amd.gemm_w8a8(st["w"], st["sw"], st["x"], st["sx"], dtype=TYPES[c["out"]])}
    if c["kind"] == "gated":
        return {"out": rt4_amd.ffn_gate_w8a8(st["w"], st["sw"], st["wu"], st["su"], st["x"], st["sx"], act=c["act"], dtype=TYPES[c["out"]])}
    if c["kind"] == "gated4":
        return {"out": rt4_amd.ffn_gate_w4a8(st["w"], st["sw"], st["wu"], st["su"], st["x"], st["sx"], act=c["act"])}
    if c["kind"] == "quant":
        q, s = rt4_amd.quant_token_a8(st["x"])
        return {"codes": q, "scale": s}
    h, n = rt4_amd.block_norm(st["h"], st["y"], weight=st["weight"], post_weight=st["post_weight"], gate=st["gate"], scale=SCALE, eps=EPS, out=c["n"])
    out = {} if st["y"] is None else {"h": h}
    return out | ({"codes": n[0], "scale": n[1]} if isinstance(n, tuple) else {"n": n})


def _act(x, name):
    if name == "silu":
        return x / (1 + (-x).exp())
    return 0.5 * x * (1 + (math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)).tanh())


def _plain_linear(st):
    c = (st["x"].float() @ st["w"].float().T) * st["sx"][:, None] * st["sw"]
    return {"out": c.to(TYPES[st["case"]["out"]])}


def _plain_gated(st):
    x = st["x"].float()
    g = (x @ st["w"].float().T) * st["sx"][:, None] * st["sw"]
    u = (x @ st["wu"].float().T) * st["sx"][:, None] * st["su"]
    return {"out": (_act(g, st["case"]["act"]) * u).to(TYPES[st["case"]["out"]])}


def _rt4_values(wq, ws):
    N = wq.shape[0]
    c = (wq[..., None] << torch.arange(28, -1, -4, dtype=torch.int32, device=wq.device)) >> 28
    return (c.reshape(N, -1, G) * ws.view(torch.float16).float()[..., None]).reshape(N, -1)


def _plain_gated4(st):
    M, K = st["x"].shape
    x = st["x"].reshape(M, K // 8, 2, 4).transpose(-1, -2).reshape(M, K // G, G).float()
    x = (x * st["sx"][..., None]).reshape(M, K)
    g, u = x @ _rt4_values(st["w"], st["sw"]).T, x @ _rt4_values(st["wu"], st["su"]).T
    return {"out": _act(g, st["case"]["act"]) * u}


def _codes_of(p, most, low):
    """Codes and maxima of 64-bit values [..., n]: the nearest integers to most * p / max|p|."""
    a = p.abs().amax(-1, keepdim=True)
    q = (p * most / torch.where(a > 0, a, torch.ones_like(a))).round_().clamp_(low, most)
    return q.to(torch.int8), a.squeeze(-1)


def _rms(x, eps):
    return 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def _plain_norm(st):
    how, h = st["case"]["n"], st["h"].double()
    out = {}
    if st["y"] is not None:
        y = st["y"].double()
        if st["post_weight"] is not None:
            y = y * _rms(y, EPS) * st["post_weight"].double()
        if st["gate"] is not None:
            y = y * st["gate"].double()
        out["h"] = (h + SCALE * y).to(st["h"].dtype)
        h = out["h"].double()                                                     # the norm sees the residual as it is stored
    r = _rms(h, EPS)
    p = h * st["weight"].double()
    if how in TYPES:
        return out | {"n": (p * r).to(TYPES[how])}
    if how == "token":
        q, a = _codes_of(p, 127, -128)
        s = a * r[:, 0] / 127
    else:
        M, K = p.shape
        most = 127 if how == "act" else 119
        q, a = _codes_of(p.reshape(M, K // G, G), most, -128)
        q = q.reshape(M, K // 8, 4, 2).transpose(-1, -2).reshape(M, K)
        s = a * r / most
        s = s if how == "act" else s.T.contiguous()
        a = a if how == "act" else a.T
    return out | {"codes": q, "scale": torch.where(a > 0, s, torch.ones_like(s)).float()}


def _plain_quant(st):
    q, a = _codes_of(st["x"].double(), 127, -128)
    return {"codes": q, "scale": torch.where(a > 0, a / 127, torch.ones_like(a)).float()}


# ------------------------------------------------------- work and 64 bits --
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}


def work(case):
    M, K, kind = case["M"], case["K"], case["kind"]
    if kind in ("linear", "gated"):
        N, n = case["N"], 2 if kind == "gated" else 1
        return {"bytes": n * N * (K + 4) + M * (K + 4) + M * N * _SIZE[case["out"]], "flops": 2 * n * M * N * K}
    if kind == "gated4":
        N = case["N"]
        return {"bytes": 2 * N * (K // 2 + K // 64) + M * (K + K // 32) + 4 * M * N, "flops": 4 * M * N * K}
    if kind == "quant":
        return {"bytes": M * K * (_SIZE[case["x"]] + 1) + 4 * M, "flops": 3 * M * K}
    with_y = case["y"] != "none"
    b = M * K * _SIZE[case["h"]] * (2 if with_y else 1) + 4 * K
    if with_y:
        b += M * K * _SIZE[case["y"]] + (4 * K if case["post"] else 0)
        b += {"none": 0, "channel": K, "token": M * K}[case["gate"]] * _SIZE[case["y"]]
    b += M * K * _SIZE[case["n"]] if case["n"] in _SIZE else M * K + 4 * M * (1 if case["n"] == "token" else K // G)
    return {"bytes": b, "flops": (12 if with_y else 6) * M * K}


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    f = torch.float64

    def act(x):
        if case["act"] == "silu":
            return x * torch.sigmoid(x)
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))    # (1 + tanh z) / 2 is the logistic function of 2 z

    if kind in ("linear", "gated"):
        x, sx = st["x"].to(f), st["sx"].to(f)[:, None]
        one = lambda w, s: torch.mm(x, w.to(f).t().contiguous()) * (sx * s.to(f))  # noqa: E731
        a = one(st["w"], st["sw"])
        return {"out": a if kind == "linear" else act(a) * one(st["wu"], st["su"])}
    if kind == "gated4":
        M, K = st["x"].shape
        at = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=DEV)                           # where elements 0..7 of a block stand
        x = st["x"].reshape(M, K // 8, 8)[:, :, at].reshape(M, K).to(f) * st["sx"].to(f).repeat_interleave(G, 1)

        def one(w, s):
            b = torch.stack([(w >> (4 * e)) & 15 for e in range(8)], -1).reshape(w.shape[0], K)
            b = torch.where(b > 7, b - 16, b).to(f) * s.view(torch.float16).to(f).repeat_interleave(G, 1)
            return torch.mm(x, b.t().contiguous())

        return {"out": act(one(st["w"], st["sw"])) * one(st["wu"], st["su"])}
    if kind == "quant":
        x = st["x"].to(f)
        a = torch.maximum(x.amax(1), -x.amin(1))
        return {"codes": None, "scale": a / 127}
    out = {}
    h = st["h"].to(f)
    if st["y"] is not None:
        y = st["y"].to(f)
        k = torch.full_like(y, SCALE)
        if st["gate"] is not None:
            k = k * st["gate"].to(f)
        if st["post_weight"] is not None:
            k = k * st["post_weight"].to(f) * torch.rsqrt((y * y).sum(1, keepdim=True) / y.shape[1] + EPS)
        out["h"] = torch.addcmul(h, k, y)
        h = out["h"].to(st["h"].dtype).to(f)
    n = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * st["weight"].to(f)
    if case["n"] in TYPES:
        return out | {"n": n}
    if case["n"] == "token":
        return out | {"codes": None, "scale": torch.linalg.vector_norm(n, math.inf, dim=1) / 127}
    s = torch.linalg.vector_norm(n.reshape(n.shape[0], -1, G), math.inf, dim=2)
    return out | {"codes": None, "scale": s / 127 if case["n"] == "act" else s.t().contiguous() / 119}
