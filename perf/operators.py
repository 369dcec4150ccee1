"""Timing cases of the operators of a draft-and-verify decode step, through rt4_amd's public functions.

Three operators over the int4-KV cache of the 27B layer shapes (24 query heads over 4 KV heads, head dim 256, vocabulary
248320) and of sizes around them:

* ``attention``: ``attention_tree``, attention of 1-64 new tokens per sequence, arranged as a tree (a chain, or one token, are
  trees too), over each sequence's cache and over the tree's own keys (a 64-key tile of the cache's format).
* ``verify``:    ``verify_tree``, which of the drafted tokens the target's logits accept, and the token that follows them.
* ``append``:    ``kv_append_rows``, new keys and values of several sequences quantized into their caches at lengths that are
  known on the device only: the draft tile, the accepted path of a tree, prompts of several lengths.

The caches' packed code words are the library's public format and every code in them is defined exactly, so they are
compared as the whole numbers that they are: equal or wrong.  Appends repeat on the same state, so their starts are chosen
for the second pass to find what the first found (no append crosses out of a tile that it began inside).
"""
from __future__ import annotations

import math
import pathlib
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
D, G, BG = 256, 128, 64


def listed():
    return [
        # One token of one sequence over a short cache: latency is what counts.
        {"name": "attn_decode_ctx1000", "kind": "attention", "B": 1, "T": 1, "kids": 1, "ctx": 1000, "ragged": False, "QH": 24, "KVH": 4},
        # The reference runtime's verify step, a token and its three drafts, over a long cache.
        {"name": "attn_chain4_ctx32k", "kind": "attention", "B": 1, "T": 4, "kids": 1, "ctx": 32701, "ragged": False, "QH": 24, "KVH": 4},
        # Four sequences of unlike lengths (one new, one idle) with trees of up to 16 nodes.
        {"name": "attn_tree16_b4", "kind": "attention", "B": 4, "T": 16, "kids": 3, "ctx": 8192, "ragged": True, "QH": 24, "KVH": 4},
        # A wide tree over the longest cache: many rows, where arithmetic counts.
        {"name": "attn_tree61_ctx131k", "kind": "attention", "B": 1, "T": 61, "kids": 4, "ctx": 131001, "ragged": False, "QH": 24, "KVH": 4},
        # A serving batch: 16 sequences with trees of 8 nodes.
        {"name": "attn_tree8_b16", "kind": "attention", "B": 16, "T": 8, "kids": 2, "ctx": 16384, "ragged": True, "QH": 24, "KVH": 4},
        # Drawing one token from one row of a small vocabulary: the smallest call.
        {"name": "verify_draw_v32000", "kind": "verify", "B": 1, "T": 1, "kids": 1, "V": 32000, "probs": False},
        # Three sampled drafts and their token, with the drafts' probabilities, over the whole vocabulary.
        {"name": "verify_chain4_probs", "kind": "verify", "B": 1, "T": 4, "kids": 1, "V": 248320, "probs": True},
        # Eight sequences with trees of top tokens, some greedy, one idle.
        {"name": "verify_tree16_b8", "kind": "verify", "B": 8, "T": 16, "kids": 3, "V": 248320, "probs": False},
        # Trees whose siblings were drawn from one distribution; an odd vocabulary.
        {"name": "verify_tree13_probs", "kind": "verify", "B": 2, "T": 13, "kids": 3, "V": 100277, "probs": True},
        # The draft tile of the verify step above.
        {"name": "append_draft4", "kind": "append", "B": 1, "T": 4, "KVH": 4, "cap": 64, "from": "zero"},
        # The accepted paths of 16 trees of 8 nodes.
        {"name": "append_path_b16", "kind": "append", "B": 16, "T": 8, "KVH": 4, "cap": 4096, "from": "path"},
        # Four prompts (or parts of them) of up to 1000 tokens.
        {"name": "append_prompt_b4", "kind": "append", "B": 4, "T": 1000, "KVH": 4, "cap": 4096, "from": "tile"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "verify", "verify", "append"])
    if kind == "attention":
        kvh = rng.choice([1, 2, 4, 8])
        T, B = _log(rng, 1, 64), _log(rng, 1, 16)
        ctx = _log(rng, 1, 131072)
        qh = kvh * rng.choice([1, 4, 6, 8])
        while B * ctx * T * qh > 131072 * 61 * 24 or B * ctx * kvh > 131072 * 4:
            ctx = 1 + ctx // 2
        return {"kind": kind, "B": B, "T": T, "kids": rng.randint(1, 4), "ctx": ctx, "ragged": rng.random() < 0.7, "QH": qh, "KVH": kvh}
    if kind == "verify":
        B, T, V = _log(rng, 1, 16), _log(rng, 1, 64), _log(rng, 500, 248320)
        while B * T * V > 8 * 16 * 248320:
            T = (T + 1) // 2
            B = (B + 1) // 2
        return {"kind": kind, "B": B, "T": T, "kids": rng.randint(1, 4), "V": V, "probs": rng.random() < 0.5}
    how = rng.choice(["zero", "path", "tile"])
    T = _log(rng, 1, 1000) if how == "tile" else _log(rng, 1, 64)
    return {"kind": kind, "B": _log(rng, 1, 16), "T": T, "KVH": rng.choice([1, 2, 4, 8]),
            "cap": 64 if how == "zero" else 64 * _log(rng, 20, 64), "from": how}


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1 + seed)
    return g


def _codes4(x, s):
    return torch.round(x / s).clamp(-8, 7).to(torch.int32)


def _pack8(c):
    """int32 codes [..., 8] -> one dword, low nibble first."""
    w = (c.to(torch.int64) & 15) << torch.arange(0, 32, 4, device=c.device)
    w = w.sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _scale7(x, dim):
    a = x.abs().amax(dim, keepdim=True)
    return torch.where(a > 0, a / torch.full_like(a, 7), torch.ones_like(a))       # (by a plain 7 torch multiplies with 1/7)


def _quant_dims(x):
    """[..., 256] -> (packed [..., 32], scales [..., 2]): K and Q, per 128 dims."""
    xg = x.unflatten(-1, (D // G, G))
    s = _scale7(xg, -1)
    return _pack8(_codes4(xg, s).flatten(-2).unflatten(-1, (D // 8, 8))), s.squeeze(-1)


def _quant_tiles(v):
    """[..., 64 n, 256] -> (packed [..., 8 n, 256], scales [..., n, 256]): V, per (64 keys, dim)."""
    vt = v.unflatten(-2, (v.shape[-2] // BG, BG))
    s = _scale7(vt, -2)
    c = _codes4(vt, s).unflatten(-2, (BG // 8, 8)).transpose(-1, -2)
    return _pack8(c).flatten(-3, -2), s.squeeze(-2)


def _cache(B, KVH, cap, g):
    """Caches of B sequences, filled with quantized N(0,1) keys and values."""
    kc = torch.empty((B, KVH, cap, D // 8), dtype=torch.int32, device=DEV)
    ksc = torch.empty((B, KVH, D // G, cap), device=DEV)
    vc = torch.empty((B, KVH, cap // 8, D), dtype=torch.int32, device=DEV)
    vsc = torch.empty((B, KVH, cap // BG, D), device=DEV)
    for b in range(B):
        for h in range(KVH):
            x = torch.randn((cap, D), device=DEV, generator=g)
            kc[b, h], s = _quant_dims(x)
            ksc[b, h] = s.T
            vc[b, h], vsc[b, h] = _quant_tiles(torch.randn((cap, D), device=DEV, generator=g))
    return kc, ksc, vc, vsc


def _trees(B, T, kids, seed):
    """parent [B][T]: chains for kids = 1, else random trees; of several sequences some end early, and the last of four or more is idle."""
    r = random.Random(seed * 7919 + 13)
    out = []
    for b in range(B):
        n = T if b == 0 else r.randint(max(1, T // 2), T)
        left = [kids] * T
        p = [-1]
        for i in range(1, n):
            q = i - 1 if kids == 1 else r.choice([j for j in range(i) if left[j] > 0])
            left[q] -= 1
            p.append(q)
        p += [-1] * (T - n)
        if B >= 4 and b == B - 1:
            p[0] = -2
        out.append(p)
    return torch.tensor(out, dtype=torch.int32)


def _up(n, m):
    return (n + m - 1) // m * m


def prepare(case, seed):
    g = _gen(seed)
    r = random.Random(seed * 31 + 5)
    B, T = case["B"], case["T"]
    st = {"case": case}
    if case["kind"] == "attention":
        QH, KVH, ctx = case["QH"], case["KVH"], case["ctx"]
        cap = _up(ctx + BG, BG)
        lens = [ctx] * B
        if case["ragged"]:
            lens = [ctx if b == 0 else 0 if b == 1 else r.randint(0, ctx) for b in range(B)]
        st["kv"] = _cache(B, KVH, cap, g)
        st["draft"] = _cache(B, KVH, BG, g)
        st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["kv_max"] = ctx
        st["parent"] = _trees(B, T, case["kids"], seed).to(DEV)
        # Heads from flat (scores of deviation 1) to sharp (5).
        q = torch.randn((B * T, QH, D), device=DEV, generator=g) / 16 * torch.linspace(1, 5, QH, device=DEV)[:, None]
        qq, qs = _quant_dims(q)
        st["qq"], st["qs"] = qq.transpose(0, 1).contiguous(), qs.permute(1, 2, 0).contiguous()
    elif case["kind"] == "verify":
        V = case["V"]
        parent = _trees(B, T, case["kids"], seed)
        at = (parent.clamp_min(0).long() + torch.arange(B)[:, None] * T).reshape(-1).to(DEV)
        logits = torch.randn((B * T, V), device=DEV, generator=g) * 2.5
        temp = torch.tensor([0.8 if b % 4 == 0 else 1.0 if b % 4 == 1 else 0.0 if b % 4 == 2 else 0.6 for b in range(B)], device=DEV)
        # The drafter sees the target's logits through noise.
        seen = logits + 0.5 * torch.randn((B * T, V), device=DEV, generator=g)
        if case["probs"]:
            t = temp.clamp_min(0.05).repeat_interleave(T)[:, None]
            q = torch.softmax(seen / t, -1)
            st["q"] = q
            draft = torch.multinomial(q[at], 1, generator=g)[:, 0]
        else:
            top = seen.topk(max(1, case["kids"]), -1).indices
            kid = torch.tensor([[p[1:i].count(p[i]) for i in range(T)] for p in parent.tolist()])
            draft = top[at, kid.reshape(-1).clamp_max(top.shape[1] - 1).to(DEV)]
            st["q"] = None
        st |= {"logits": logits, "draft": draft.reshape(B, T).to(torch.int32), "parent": parent.to(DEV), "temp": temp}
        st["u"] = torch.rand((B, T), device=DEV, generator=g)
    else:
        KVH, cap, how = case["KVH"], case["cap"], case["from"]
        st["kv"] = _cache(B, KVH, cap, g) if how != "zero" else (
            torch.zeros((B, KVH, cap, D // 8), dtype=torch.int32, device=DEV), torch.ones((B, KVH, D // G, cap), device=DEV),
            torch.zeros((B, KVH, cap // 8, D), dtype=torch.int32, device=DEV), torch.ones((B, KVH, cap // BG, D), device=DEV))
        st["stage"] = None if how == "zero" else torch.randn((B, KVH, BG, D), device=DEV, generator=g)
        st["kf"] = torch.randn((B, T, KVH, D), device=DEV, generator=g)
        st["vf"] = torch.randn((B, T, KVH, D), device=DEV, generator=g)
        st["rows"] = st["count"] = st["kv_len"] = None
        if how != "zero":
            count = [T if b == 0 else r.randint(1, T) for b in range(B)]
            start = [BG * r.randint(0, (cap - T) // BG - 1) + (r.randint(0, BG - T) if how == "path" else 0) for b in range(B)]
            st["count"] = torch.tensor(count, dtype=torch.int32, device=DEV)
            st["kv_len"] = torch.tensor([s + n for s, n in zip(start, count)], dtype=torch.int32, device=DEV)
        if how == "path":
            rows = [sorted(r.sample(range(T), n)) + [-1] * (T - n) for n in count]
            st["rows"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------------------ passes --
def run(state):
    if own:
        return _run_own(state)
    return {"attention": _plain_attention, "verify": _plain_verify, "append": _plain_append}[state["case"]["kind"]](state)


_pkg = str(pathlib.Path(__file__).resolve().parents[1] / "k100lc-rt4_amd")


def _run_own(st):
    if "rt4_amd" not in sys.modules and _pkg not in sys.path:
        sys.path.insert(0, _pkg)
    import rt4_amd
    kind = st["case"]["kind"]
    if kind == "attention":
        return {"out": rt4_amd.attention_tree(st["qq"], st["qs"], *st["kv"], st["kv_len"], *st["draft"], st["parent"],
                                              ratio=st["case"]["QH"] // st["case"]["KVH"], kv_max=st["kv_max"])}
    if kind == "verify":
        tokens, path, count = rt4_amd.verify_tree(st["logits"], st["draft"], st["parent"], st["u"], temp=st["temp"], draft_probs=st["q"],
                                                  max_children=st["case"]["kids"] if st["q"] is not None else None)
        return {"tokens": tokens, "path": path, "count": count}
    rt4_amd.kv_append_rows(*st["kv"], st["stage"], st["kf"], st["vf"], kv_len=st["kv_len"], rows=st["rows"], count=st["count"])
    return _appended(st)


def _appended(st):
    out = dict(zip(("kc", "ksc", "vc", "vsc"), st["kv"]))
    if st["stage"] is not None:
        out["stage"] = st["stage"]
    return out


def _unpack8(w):
    """int32 [...] -> codes [..., 8]."""
    return (w[..., None] << torch.arange(28, -1, -4, dtype=torch.int32, device=w.device)) >> 28


def _values(kc, ksc, vc, vsc):
    """The values that caches [B, KVH, ...] stand for: K and V f32 [B, KVH, cap, 256]."""
    k = (_unpack8(kc).flatten(-2).unflatten(-1, (D // G, G)) * ksc.transpose(-1, -2)[..., None]).flatten(-2)
    v = _unpack8(vc).transpose(-1, -2).flatten(-3, -2)
    return k, (v.unflatten(-2, (v.shape[-2] // BG, BG)) * vsc[..., None, :]).flatten(-3, -2)


def _ancestors(parent):
    """f32 [B, T, T]: whether node j is node i or above it, with no row for nodes that hang under no root."""
    T = parent.shape[1]
    i = torch.arange(T, device=parent.device)
    up = ((parent[:, :, None] == i) & (i < i[:, None])).float() + torch.eye(T, device=parent.device)
    two = lambda a: (a @ a > 0).float()  # noqa: E731
    a = two(two(two(two(two(two(up))))))
    return a * a[:, :, :1] * (parent[:, :1, None] == -1)


def _plain_attention(st):
    B, T = st["parent"].shape
    KVH = st["kv"][0].shape[1]
    R = st["case"]["QH"] // KVH
    q = (_unpack8(st["qq"]).flatten(-2).unflatten(-1, (D // G, G)) * st["qs"].transpose(-1, -2)[..., None]).flatten(-2)   # [QH, B T, D]
    q = q.reshape(KVH, R, B, T, D).permute(2, 0, 1, 3, 4).reshape(B, KVH, R * T, D)
    sees = _ancestors(st["parent"]) > 0
    cap = st["kv"][0].shape[2]
    k, v = _values(*st["kv"])
    kd, vd = _values(*st["draft"])
    s = torch.cat([q @ k.transpose(-1, -2).contiguous(), q @ kd.transpose(-1, -2).contiguous()], -1)
    live = sees[:, :, 0]
    prefix = (torch.arange(cap, device=q.device) < st["kv_len"][:, None])[:, None] & live[:, :, None]
    tail = torch.zeros((B, T, BG - T), dtype=torch.bool, device=q.device)
    mask = torch.cat([prefix, sees, tail], -1)[:, None, None].expand(B, KVH, R, T, cap + BG).reshape(B, KVH, R * T, cap + BG)
    s = s.masked_fill_(~mask, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    o = p[..., :cap] @ v + p[..., cap:] @ vd
    o = o / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return {"out": o.reshape(B, KVH, R, T, D).permute(1, 2, 0, 3, 4).reshape(KVH * R, B * T, D)}


def _plain_verify(st):
    parent, draft, u, q = st["parent"], st["draft"].long(), st["u"].double(), st["q"]
    B, T = parent.shape
    V = st["logits"].shape[-1]
    temp = st["temp"].double()[:, None]
    x = st["logits"].double().view(B, T, V) / torch.where(temp > 0, temp, torch.ones_like(temp))[..., None]
    m = x.amax(-1, keepdim=True)
    top = x.argmax(-1)
    p = (x - m).exp()
    p = p / p.sum(-1, keepdim=True)
    q = None if q is None else q.double().view(B, T, V)
    i = torch.arange(T, device=parent.device)
    anc = _ancestors(parent)
    live = anc[:, :, 0] > 0
    up = parent.clamp_min(0).long()
    sib = (parent[:, :, None] == parent[:, None, :]) & (i < i[:, None]) & live[:, :, None] & live[:, None, :] & (i > 0)   # earlier sibling j of node i
    seq = torch.arange(B, device=parent.device)[:, None]
    pc = p[seq, up, draft]
    if q is None:
        first = ~(sib & (draft[:, :, None] == draft[:, None, :])).any(-1)          # the first sibling with its token
        W = 1 - (sib & first[:, None, :]).double().mul(pc[:, None, :]).sum(-1)
        yes = (u * W < pc) & first
        a = rank = None
    else:
        rank = sib.sum(-1)
        kmax = st["case"]["kids"]
        a, W = torch.zeros((B, T, kmax + 1), dtype=torch.float64, device=p.device), torch.ones((B, T, kmax + 1), dtype=torch.float64, device=p.device)
        for k in range(kmax):
            a[..., k + 1] = a[..., k] + W[..., k]
            W[..., k + 1] = (p - a[..., k + 1, None] * q).clamp_min(0).sum(-1) if k + 1 < kmax else 1
        qc = q[seq, up, draft]
        yes = u * W[seq, up, rank] * qc < pc - a[seq, up, rank] * qc
    yes = torch.where(temp > 0, yes, draft == top[seq, up])
    # A node is on the path when it and all above it (but the root) are accepted and no sibling before one of them was.
    ok = yes & ~(sib & yes[:, None, :]).any(-1)
    on = live & ~((anc > 0) & ~ok[:, None, :] & (i > 0)).any(-1)
    count = on.sum(-1)
    pos = on.long().cumsum(-1) - 1
    path = torch.full((B, T + 1), -1, dtype=torch.int64, device=parent.device).scatter(1, torch.where(on, pos, T), i.expand(B, T))[:, :T]
    last = path.amax(-1).clamp_min(0)[:, None]
    w = p[seq, last][:, 0]
    kid = (parent == last) & live & (i > 0)
    if q is None:
        w = w.scatter(1, torch.where(kid, draft, V - 1), torch.where(kid, torch.zeros_like(pc), w[:, V - 1:]))
        w[:, V - 1:] *= ~(kid & (draft == V - 1)).any(-1, keepdim=True)
    else:
        w = (w - a[seq, last, kid.sum(-1, keepdim=True)] * q[seq, last][:, 0]).clamp_min(0)
    c = w.cumsum(-1)
    drawn = (c > u[:, :1] * c[:, -1:]).long().argmax(-1)
    drawn = torch.where(temp[:, 0] > 0, drawn, top[seq, last][:, 0])
    tokens = torch.full((B, T + 1), -1, dtype=torch.int64, device=parent.device)
    tokens = tokens.scatter(1, torch.where(on & (i > 0), pos - 1, T), draft)
    tokens = tokens.scatter(1, torch.where(count > 0, count - 1, T)[:, None], drawn[:, None])[:, :T]
    return {"tokens": tokens.int(), "path": path.int(), "count": count.int()}


def _plain_append(st):
    kc, ksc, vc, vsc = st["kv"]
    stage, kf, vf = st["stage"], st["kf"], st["vf"]
    B, T, KVH = kf.shape[:3]
    dev = kf.device
    n = torch.full((B,), T, device=dev) if st["count"] is None else st["count"].long()
    start = torch.zeros_like(n) if st["kv_len"] is None else st["kv_len"].long() - n
    seq = torch.arange(B, device=dev)[:, None]
    j = torch.arange(T, device=dev).expand(B, T)
    j = torch.where(j < n[:, None], j, torch.zeros_like(j))                # rows after the last repeat the first
    row = j if st["rows"] is None else st["rows"].long().gather(1, j)
    codes, s = _quant_dims(kf[seq, row])                                    # [B, T, KVH, ..]
    key = start[:, None] + j
    kc[seq, :, key] = codes
    ksc.permute(0, 3, 1, 2)[seq, key] = s
    # Touched tiles (those after the last repeat it), each with its 64 slots.
    tile = torch.arange((T + BG - 2) // BG + 1, device=dev)
    tile = torch.minimum(start[:, None] // BG + tile, (start + n - 1)[:, None] // BG)
    at = tile[:, :, None] * BG + torch.arange(BG, device=dev)              # [B, tiles, 64] keys
    back = (at - start[:, None, None]).clamp(0, T - 1)
    src = back if st["rows"] is None else st["rows"].long().clamp_min(0)[:, None].expand(B, tile.shape[1], T).gather(2, back)
    fresh = ((at >= start[:, None, None]) & (at < (start + n)[:, None, None]))[..., None, None]
    x = torch.where(fresh, vf[seq[..., None], src], torch.zeros((), device=dev))
    if stage is not None:
        x = torch.where((at < start[:, None, None])[..., None, None], stage.transpose(1, 2)[:, None], x)
    codes, s = _quant_tiles(x.permute(0, 3, 1, 2, 4).flatten(2, 3))        # [B, KVH, 8 tiles, D], [B, KVH, tiles, D]
    if stage is not None:
        k = torch.arange(BG, device=dev) + ((start + n - 1) // BG * BG)[:, None]
        k = torch.where(k < (start + n)[:, None], k, k - BG)               # the last tile's keys, beneath them the tile before's
        back = (k - start[:, None]).clamp(0, T - 1)
        src = back if st["rows"] is None else st["rows"].long().clamp_min(0).gather(1, back)
        new = torch.where((k >= start[:, None])[..., None, None], vf[seq, src], stage.transpose(1, 2))
        stage.copy_(new.transpose(1, 2))
    vc.unflatten(2, (vc.shape[2] // 8, 8))[seq, :, tile] = codes.unflatten(2, (tile.shape[1], 8)).transpose(1, 2)
    vsc[seq, :, tile] = s.transpose(1, 2)
    return _appended(st)


# -------------------------------------------------------------------- work --
def work(case):
    B, T = case["B"], case["T"]
    if case["kind"] == "attention":
        QH, KVH = case["QH"], case["KVH"]
        keys = case["ctx"] * (B if not case["ragged"] else max(1.0, 1 + max(0, B - 2) / 2))       # ragged lengths average half
        cache = KVH * (2 * D // 2 + 4 * D // G + 4 * D / BG)
        io = B * T * QH * (D / 2 + 8 + 4 * D) + B * KVH * T * (D + 8) + B * KVH * 4 * D
        return {"bytes": keys * cache + io, "flops": 4.0 * T * QH * D * (keys + B * T / 2)}
    if case["kind"] == "verify":
        rows = B * T
        return {"bytes": 4.0 * rows * case["V"] * (2 if case["probs"] else 1) + 20.0 * rows, "flops": 4.0 * rows * case["V"]}
    rows = B * (T if case["from"] == "zero" else T / 2)
    tiles = B * (1 if case["from"] != "tile" else T / 128 + 1)
    staged = 0 if case["from"] == "zero" else 4.0 * B * case["KVH"] * D * min(BG, 32 + T)
    return {"bytes": case["KVH"] * (rows * (8 * D + D / 2 + 8) + tiles * (BG / 8 * 4 * D + 4 * D)) + staged, "flops": 6.0 * rows * case["KVH"] * D}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "verify": _exact_verify, "append": _exact_append}[case["kind"]](st)


def _chain(parent, i):
    """The nodes from i up to the root, or none where i hangs under no root."""
    up = [i]
    while i > 0:
        p = parent[i]
        if not 0 <= p < i:
            return []
        i = p
        up.append(i)
    return up if parent[0] == -1 else []


def _nib64(w):
    return torch.stack([((w >> (4 * e)) & 15) for e in range(8)], -1).add(8).remainder(16).sub(8).double()


def _exact_attention(st):
    parent = st["parent"].tolist()
    lens = st["kv_len"].tolist()
    B, T = len(parent), len(parent[0])
    KVH = st["kv"][0].shape[1]
    QH = st["case"]["QH"]
    R = QH // KVH
    out = torch.zeros((QH, B * T, D), dtype=torch.float64, device=DEV)
    for b in range(B):
        n = lens[b]
        sees = torch.zeros((T, BG), dtype=torch.bool, device=DEV)
        for i in range(T):
            for j in _chain(parent[b], i):
                sees[i, j] = True
        rows = [i for i in range(T) if _chain(parent[b], i)]
        if not rows:
            continue
        for h in range(KVH):
            ks, vs = [], []
            for (kc, ksc, vc, vsc), keys in ((st["kv"], (n + BG - 1) // BG * BG), (st["draft"], BG)):
                k = _nib64(kc[b, h, :keys]).reshape(keys, D)
                ks.append(k * ksc[b, h, :, :keys].double().repeat_interleave(G, 0).T)
                v = _nib64(vc[b, h, :keys // 8]).transpose(1, 2).reshape(keys, D)
                vs.append(v * vsc[b, h, :keys // BG].double().repeat_interleave(BG, 0))
            K, Vv = torch.cat([ks[0][:n], ks[1]]), torch.cat([vs[0][:n], vs[1]])
            for r in range(h * R, (h + 1) * R):
                at = [b * T + i for i in rows]
                q = _nib64(st["qq"][r, at]).reshape(len(at), D) * st["qs"][r][:, at].double().repeat_interleave(G, 0).T
                s = q @ K.T.contiguous()
                s[:, n:] = s[:, n:].masked_fill(~sees[rows], -math.inf)
                out[r, at] = torch.softmax(s, -1) @ Vv
    return {"out": out}


def _exact_verify(st):
    parent, draft = st["parent"].tolist(), st["draft"].tolist()
    u, temp = st["u"].double().tolist(), st["temp"].double().tolist()
    B, T = len(parent), len(parent[0])
    V = st["logits"].shape[-1]
    tokens, path, count = (np.full(s, -1, np.int32) for s in ((B, T), (B, T), (B,)))
    for b in range(B):
        if parent[b][0] != -1:
            count[b] = 0
            continue
        node, n, i = 0, 1, 0
        path[b, 0] = 0
        while True:
            x = st["logits"][b * T + node].double().cpu().numpy()
            q = None if st["q"] is None else st["q"][b * T + node].double().cpu().numpy()
            best = int(np.argmax(x))
            left = np.exp((x - x.max()) / (temp[b] or 1.0))
            left /= left.sum()
            took = None
            for c in range(node + 1, T):
                if parent[b][c] != node:
                    continue
                t = draft[b][c]
                if temp[b] <= 0:
                    took = c if t == best else None
                elif q is None:
                    took = c if u[b][c] * left.sum() < left[t] else None
                    if took is None:
                        left[t] = 0.0
                else:
                    took = c if u[b][c] * q[t] < left[t] else None
                    if took is None:
                        left = np.maximum(left - q, 0.0)
                        left /= left.sum()
                if took is not None:
                    break
            if took is None:
                break
            tokens[b, n - 1], path[b, n] = draft[b][took], took
            node, n = took, n + 1
        c = np.cumsum(left)
        tokens[b, n - 1] = best if temp[b] <= 0 else int(np.searchsorted(c, u[b][0] * c[-1], side="right"))
        count[b] = n
    return {"tokens": tokens, "path": path, "count": count}


def _exact_append(st):
    """Codes by numpy's IEEE float32 quotients, which the format names; the scales and the stage in 64 bits."""
    kc, ksc, vc, vsc = (x.cpu().numpy().copy() for x in st["kv"])
    ksc, vsc = ksc.astype(np.float64), vsc.astype(np.float64)
    stage = None if st["stage"] is None else st["stage"].cpu().numpy().copy()
    kf, vf = st["kf"].cpu().numpy(), st["vf"].cpu().numpy()
    B, T, KVH = kf.shape[:3]

    def quant(x):                                   # [n, ...]: one scale over axis 0
        a = np.abs(x).max(0)
        s = np.where(a > 0, a / np.float32(7), np.float32(1)).astype(np.float32)
        return np.clip(np.rint((x / s).astype(np.float32)), -8, 7).astype(np.int64), np.where(a > 0, a.astype(np.float64) / 7, 1.0)

    def words(c):                                   # [8, ...] -> int32
        w = sum((c[e] & 15) << (4 * e) for e in range(8))
        return w.astype(np.uint32).view(np.int32)

    for b in range(B):
        n = T if st["count"] is None else int(st["count"][b])
        s0 = 0 if st["kv_len"] is None else int(st["kv_len"][b]) - n
        rows = list(range(n)) if st["rows"] is None else st["rows"][b, :n].tolist()
        for j, r in enumerate(rows):
            c, s = quant(kf[b, r].reshape(KVH, 2, G).transpose(2, 0, 1))            # [128, KVH, 2]
            ksc[b, :, :, s0 + j] = s
            kc[b, :, s0 + j] = words(c.transpose(1, 2, 0).reshape(KVH, D // 8, 8).transpose(2, 0, 1).copy())
        old = None if stage is None else stage[b].copy()
        for t in range(s0 // BG, (s0 + n - 1) // BG + 1):
            x = np.zeros((BG, KVH, D), np.float32)
            for k in range(BG):
                key = t * BG + k
                if key < s0:
                    x[k] = old[:, k]
                elif key < s0 + n:
                    x[k] = vf[b, rows[key - s0]]
                    if stage is not None:
                        stage[b][:, k] = x[k]
            c, s = quant(x)
            vsc[b, :, t] = s
            vc[b, :, 8 * t:8 * t + 8] = words(c.reshape(8, 8, KVH, D).transpose(1, 2, 0, 3).copy())
    out = {"kc": kc, "ksc": ksc, "vc": vc, "vsc": vsc}
    if stage is not None:
        out["stage"] = stage.astype(np.float64)
    return out
