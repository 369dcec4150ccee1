"""Draft-and-verify decode steps: row appends at device lengths, tree attention, verification.

Expectations are plain numpy: the appends are bit-exact against the oracle's single-sequence appends of the same rows
(oracle/rt4_oracle.c), the attention is a 64-bit softmax over the values that the codes stand for, the verification a
literal walk in 64 bits whose tokens and paths have to be equal.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

D, BG, G = 256, 64, 128


# ------------------------------------------------------------ expectations --
def nibbles(w):
    nib = (np.asarray(w).view(np.uint32)[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    return np.where(nib >= 8, nib.astype(np.int64) - 16, nib.astype(np.int64))


def chain(parent, i):
    """Node i and those above it up to the root; nothing where it hangs under no root."""
    up = [i]
    while i > 0:
        p = int(parent[i])
        if not 0 <= p < i:
            return []
        i = p
        up.append(i)
    return up if parent[0] == -1 else []


def cache_values(kc, ksc, vc, vsc):
    """64-bit K, V [cap, 256] of one sequence's KV head."""
    cap = kc.shape[0]
    K = nibbles(kc).reshape(cap, D) * np.repeat(ksc.astype(np.float64).T, G, axis=1)
    V = nibbles(vc).transpose(0, 2, 1).reshape(cap, D) * np.repeat(vsc.astype(np.float64), BG, axis=0)
    return K, V


def tree_attention(qq, qs, kv, lens, draft, parent, ratio):
    """(out f64 [QH, B*T, D], error bound f64 of the same shape).

    The bound counts fp32 roundings (half a step, 2^-24): a score is a sum of two terms of at most three products each, in
    log2 units, 8 roundings of at most S = sum of |terms|, which moves P by as much times ln 2; exp2, the products and the
    sums within a 64-key tile and over the tiles add 160 + tiles; P may be held as two fp16 parts, 2^-22 of itself and 2^-32
    of the row's largest per key.  All of it is relative to the largest |V|."""
    QH, TP, _ = qq.shape
    B, T = parent.shape
    H = QH // ratio
    out = np.zeros((QH, B * T, D))
    tol = np.zeros((QH, B * T, 1))
    with np.errstate(invalid="ignore", over="ignore"):
        for b in range(B):
            for h in range(H):
                n = int(np.clip(lens[b], 0, kv[0].shape[2])) if kv is not None else 0
                Kd, Vd = cache_values(*(x[b, h] for x in draft))
                K, V = Kd[:0], Vd[:0]
                if n:
                    K, V = cache_values(*(x[b, h] for x in kv))
                for i in range(T):
                    see = chain(parent[b], i)
                    if not see:
                        continue
                    Ka, Va = np.concatenate([K[:n], Kd[see]]), np.concatenate([V[:n], Vd[see]])
                    for r in range(h * ratio, (h + 1) * ratio):
                        row = b * T + i
                        q = nibbles(qq[r, row]).reshape(D) * np.repeat(qs[r, :, row].astype(np.float64), G)
                        s = Ka @ q
                        S = (np.abs(Ka[:, :G] @ q[:G]) + np.abs(Ka[:, G:] @ q[G:])).max() * 1.4427
                        p = np.exp(s - s.max())
                        out[r, row] = p @ Va / p.sum()
                        tol[r, row] = np.abs(Va).max() * ((8 * S + 168 + n / BG) * 2.0**-24 + 2.0**-22 + len(s) * 2.0**-32)
    return out, tol


def verify(logits, draft, parent, u, temp, q=None, max_children=None):
    """The walk, literally, in 64 bits: (tokens, path, count)."""
    B, T = parent.shape
    V = logits.shape[1]
    tokens, path, count = np.full((B, T), -1), np.full((B, T), -1), np.zeros(B, int)
    for b in range(B):
        if parent[b, 0] != -1:
            continue
        node, n = 0, 1
        path[b, 0] = 0
        t = float(temp[b])
        while True:
            x = logits[b * T + node].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            m = x.max()
            best = int(np.argmax(x)) if m > -np.inf else -1
            w = np.zeros(V)
            if t > 0 and m > -np.inf:
                with np.errstate(invalid="ignore"):
                    w = np.where(x == m, 1.0, np.exp((x - m) / t))
                w = w / w.sum()
            qn = None if q is None else q[b * T + node].astype(np.float64)
            took, tried = None, 0
            for c in range(node + 1, T):
                if parent[b, c] != node:
                    continue
                tk = int(draft[b, c])
                real = 0 <= tk < V
                tried += 1
                if q is not None and tried > max_children:
                    continue
                if not t > 0:
                    hit = real and tk == best
                elif q is None:
                    hit = real and float(u[b, c]) * w.sum() < w[tk]
                    if not hit and real:
                        w[tk] = 0.0
                else:
                    hit = real and float(u[b, c]) * qn[tk] < w[tk]
                    if not hit:
                        w = np.maximum(w - qn, 0.0)
                        w = w / (w.sum() or 1.0)
                if hit:
                    took = c
                    break
            if took is None:
                break
            tokens[b, n - 1], path[b, n] = draft[b, took], took
            node, n = took, n + 1
        c = np.cumsum(w)
        tokens[b, n - 1] = int(np.argmax(c > float(u[b, 0]) * c[-1])) if t > 0 and c[-1] > 0 else best
        count[b] = n
    return tokens, path, count


def random_tree(rng, T, kids):
    left, p = [kids] * T, [-1]
    for i in range(1, T):
        j = i - 1 if kids == 1 else int(rng.choice([j for j in range(i) if left[j] > 0]))
        left[j] -= 1
        p.append(j)
    return p


# ---------------------------------------------------------------- CPU side --
def test_residual_law():
    """Proposals drawn from q and tested so leave the target's distribution, for one child and for two siblings."""
    rng = np.random.default_rng(5)
    V, N = 4, 2000
    p, q = rng.dirichlet(np.ones(V)), rng.dirichlet(np.ones(V)).astype(np.float32)
    q = q.astype(np.float64)
    logits = np.log(np.stack([p] * 3)).astype(np.float32)
    pt = np.exp(logits[0].astype(np.float64))
    pt /= pt.sum()
    grid = ((np.arange(N) + 0.5) / N).astype(np.float32)
    law = np.zeros(V)
    for x in range(V):                                  # one child of token x, then its residual
        acc = min(1.0, pt[x] / q[x])
        law[x] += q[x] * acc
        res = np.maximum(pt - q, 0)
        law += q[x] * (1 - acc) * res / res.sum()
    assert np.allclose(law, pt, atol=1e-12)
    # the walk above accepts that share of a grid of uniforms, and the second sibling the share of its residual
    par = np.array([[-1, 0, 0]])
    for x in range(V):
        for y in range(V):
            res = np.maximum(pt - q, 0)
            res /= res.sum()
            a1, a2 = min(1.0, pt[x] / q[x]), min(1.0, res[y] / q[y])
            got = [0, 0]
            for k in range(0, N, 10):
                _, path, n = verify(logits, np.array([[0, x, y]]), par, np.array([[0.5, grid[k], grid[k]]]), [1.0],
                                    np.stack([q] * 3), 2)
                if n[0] > 1:
                    got[path[0, 1] - 1] += 10 / N
            assert abs(got[0] - a1) <= 10 / N + 1e-6
            assert abs(got[1] - max(0.0, a2 - a1)) <= 20 / N + 1e-6


DUMMY = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


def test_append_refusals(rt4):
    L = rt4.lib()

    def call(kc=DUMMY, stage=DUMMY, kv_len=DUMMY, B=1, T=4, H=2, cap=128):
        return L.rt4_kv_append_rows(kc, DUMMY, DUMMY, DUMMY, stage, DUMMY, DUMMY, kv_len, None, None, B, T, H, cap, None)
    assert call(kc=None) == 2 and "null" in L.rt4_last_error().decode()
    assert call(stage=None) == 2 and "stage" in L.rt4_last_error().decode()
    assert call(kc=ctypes.c_void_p(0x1002)) == 2 and "misaligned" in L.rt4_last_error().decode()
    for bad in (dict(B=0), dict(B=65536), dict(T=0), dict(H=0), dict(cap=0), dict(cap=100), dict(cap=1 << 24), dict(T=129)):
        assert call(**bad) == 1 and "rt4_kv_append_rows" in L.rt4_last_error().decode(), bad


def test_attention_refusals(rt4):
    L = rt4.lib()

    def call(out=DUMMY, kc=DUMMY, kv_len=DUMMY, B=1, T=4, TP=4, QH=4, ratio=2, cap=128, kv_max=100, splits=0):
        return L.rt4_attention_tree(out, DUMMY, DUMMY, kc, DUMMY, DUMMY, DUMMY, kv_len, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, B, T,
                                    TP, QH, ratio, cap, kv_max, splits, None)
    assert call(out=None) == 2 and call(kc=None) == 2
    assert call(out=ctypes.c_void_p(0x1004)) == 2 and "misaligned" in L.rt4_last_error().decode()
    assert call(splits=-1) == 2 and call(splits=129) == 2
    for bad in (dict(B=0), dict(T=0), dict(T=65, TP=65), dict(TP=3), dict(B=2, TP=7), dict(QH=0), dict(ratio=0), dict(ratio=3),
                dict(cap=0), dict(cap=96), dict(cap=1 << 24), dict(kv_max=129), dict(kv_max=-1)):
        assert call(**bad) == 1 and "rt4_attention_tree" in L.rt4_last_error().decode(), bad


def test_verify_refusals(rt4):
    L = rt4.lib()

    def call(logits=DUMMY, q=None, ldl=100, ldq=100, B=1, T=4, V=100, kids=0):
        return L.rt4_verify_tree(DUMMY, DUMMY, DUMMY, None, logits, ldl, DUMMY, DUMMY, DUMMY, None, q, ldq, B, T, V, kids, None)
    assert call(logits=None) == 2
    assert call(logits=ctypes.c_void_p(0x1001)) == 2
    for bad in (dict(B=0), dict(T=0), dict(T=65), dict(V=0), dict(V=(1 << 22) + 1, ldl=1 << 23), dict(ldl=99), dict(B=20000),
                dict(q=DUMMY, kids=0), dict(q=DUMMY, kids=1, ldq=99)):
        assert call(**bad) == 1 and "rt4_verify_tree" in L.rt4_last_error().decode(), bad


def test_python_refusals(rt4):
    """Tensors off the device, of another type or shape never reach the library."""
    import torch
    f, i = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    try:
        torch.cuda.current_device()
    except Exception:                                   # no device here: the wrappers ask for it first
        with pytest.raises(Exception):
            rt4.verify_tree(f(4, 10), i(1, 4), i(1, 4), f(1, 4))
        return
    with pytest.raises(rt4.RT4Error):
        rt4.verify_tree(f(4, 10), i(1, 4), i(1, 4), f(1, 4))


# ---------------------------------------------------------------- GPU side --
def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    if a.dtype == np.int64:
        a = a.astype(np.int32)
    return torch.from_numpy(a).cuda()


def host(t):
    return t.cpu().numpy()


def blank_cache(rng, B, H, cap):
    """A cache whose contents are recognizable garbage."""
    return [rng.integers(0, 2**32, (B, H, cap, D // 8), dtype=np.uint32), rng.random((B, H, 2, cap), np.float32),
            rng.integers(0, 2**32, (B, H, cap // 8, D), dtype=np.uint32), rng.random((B, H, cap // BG, D), np.float32)]


def append_expected(orc, kv, stage, kf, vf, start, rows, count):
    """The oracle's appends of the chosen rows, sequence by sequence, in place."""
    B, T, H, _ = kf.shape
    cap = kv[0].shape[2]
    for b in range(B):
        n = int(np.clip(count[b], 0, T))
        if n == 0 or start[b] < 0 or start[b] + n > cap:
            continue
        sel = [int(r) for r in rows[b][:n]]
        pick = lambda x: np.stack([x[b, r] if 0 <= r < T else np.zeros_like(x[b, 0]) for r in sel])  # noqa: E731
        orc.kv_append_k(kv[0][b], kv[1][b], pick(kf), int(start[b]))
        st = stage[b] if stage is not None else np.zeros((H, BG, D), np.float32)
        orc.kv_append_v(kv[2][b], kv[3][b], st, pick(vf), int(start[b]), cap)


APPENDS = [
    # B, T, H, cap, starts, counts (None: all), rows chosen
    (1, 1, 1, 64, [0], None, False),
    (1, 1, 2, 128, [63], None, False),
    (1, 1, 2, 128, [64], None, False),
    (1, 1, 2, 128, [127], None, False),
    (3, 4, 2, 192, [61, 62, 188], [4, 2, 4], True),
    (5, 8, 2, 256, [60, 0, 250, -3, 10], [8, 0, 8, 4, -1], True),       # full path, none, past the end, before it, negative count
    (2, 64, 1, 256, [1, 63], [64, 63], True),
    (2, 65, 3, 256, [63, 191], [65, 65], False),
    (4, 300, 2, 512, [0, 64, 129, 212], [300, 1, 299, 300], False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,cap,start,count,chosen", APPENDS)
def test_append_rows(rt4, torch_gpu, orc, B, T, H, cap, start, count, chosen):
    print(f"case append B={B} T={T} H={H} cap={cap} start={start} count={count}", flush=True)
    rng = np.random.default_rng(B * 1000 + T)
    kv = blank_cache(rng, B, H, cap)
    stage = rng.standard_normal((B, H, BG, D)).astype(np.float32)
    kf, vf = (rng.standard_normal((B, T, H, D)).astype(np.float32) for _ in range(2))
    kf[0, 0, 0, :G] = 0                                 # a group of zeros: scale 1
    vf[:, :, 0, 5] = 0
    kf[-1, -1] *= 1e30
    cnt = np.full(B, T) if count is None else np.array(count)
    rows = np.tile(np.arange(T), (B, 1))
    if chosen:
        rows = np.stack([rng.permutation(T) for _ in range(B)])
        rows[0, T // 2] = rows[0, 0]                    # the same row twice
        rows[-1, 0] = T                                 # names no row: zeros
    kv_len = np.array(start) + cnt
    got = [dev(x) for x in (*kv, stage)]
    rt4.kv_append_rows(*got, dev(kf), dev(vf), kv_len=dev(kv_len), rows=dev(rows) if chosen else None,
                       count=None if count is None else dev(cnt))
    append_expected(orc, kv, stage, kf, vf, kv_len - cnt, rows, cnt)
    for name, g, w in zip(("kc", "ksc", "vc", "vsc", "stage"), got, (*kv, stage)):
        assert np.array_equal(host(g).view(np.uint32), w.view(np.uint32)), name


@pytest.mark.gpu
@pytest.mark.parametrize("T,count,with_stage", [(1, None, False), (7, [7, 3], False), (64, [64, 1], False), (64, [0, 63], True)])
def test_append_draft_tile(rt4, torch_gpu, orc, T, count, with_stage):
    print(f"case draft tile T={T} count={count}", flush=True)
    rng = np.random.default_rng(T)
    B, H = 2, 3
    kv = blank_cache(rng, B, H, BG)
    stage = rng.standard_normal((B, H, BG, D)).astype(np.float32)
    kf, vf = (rng.standard_normal((B, T, H, D)).astype(np.float32) for _ in range(2))
    got = [dev(x) for x in (*kv, stage)]
    rt4.kv_append_rows(*got[:4], got[4] if with_stage else None, dev(kf), dev(vf), count=None if count is None else dev(np.array(count)))
    cnt = np.full(B, T) if count is None else np.array(count)
    append_expected(orc, kv, stage if with_stage else None, kf, vf, np.zeros(B, int), np.tile(np.arange(T), (B, 1)), cnt)
    for name, g, w in zip(("kc", "ksc", "vc", "vsc", "stage"), got, (*kv, stage)):
        assert np.array_equal(host(g).view(np.uint32), w.view(np.uint32)), name


def attention_case(orc, rng, B, T, H, ratio, cap, sharp, TP=None):
    QH, TP = H * ratio, TP or B * T
    q = rng.standard_normal((B * T, QH, D)).astype(np.float32) * np.float32(sharp / 16)
    qq, qs = orc.attn_q_quant(q, TP)

    def cache(n):
        kv = blank_cache(rng, B, H, n)
        for b in range(B):
            orc.kv_append_k(kv[0][b], kv[1][b], rng.standard_normal((n, H, D)).astype(np.float32), 0)
            orc.kv_append_v(kv[2][b], kv[3][b], np.zeros((H, BG, D), np.float32), rng.standard_normal((n, H, D)).astype(np.float32), 0, n)
        return kv
    return qq, qs, cache(cap), cache(BG)


def spoil_unseen(kv, draft, lens, T):
    """Infinities and NaN wherever no node may look."""
    for b, n in enumerate(lens):
        n = int(np.clip(n, 0, kv[0].shape[2]))
        kv[1][b, :, :, n:] = np.nan
        kv[1][b, :, 1, n:] = np.inf
        kv[3][b, :, (n + BG - 1) // BG:] = np.nan
    draft[1][:, :, :, T:] = np.nan


def check_attention(out, want, tol):
    err = np.abs(host(out).astype(np.float64)[:, :want.shape[1]] - want)
    assert np.isfinite(err).all()
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()


ATTENTIONS = [
    # B, T, kids, H, ratio, cap, lengths, score deviation
    (1, 1, 1, 1, 1, 64, [0], 1),
    (1, 1, 1, 1, 1, 64, [1], 1),
    (1, 1, 1, 2, 6, 64, [64], 2),
    (2, 1, 1, 2, 6, 192, [65, 127], 5),
    (1, 2, 1, 1, 8, 128, [63], 1),
    (3, 4, 1, 2, 6, 320, [0, 257, 320], 3),
    (1, 5, 2, 1, 3, 1024, [1000], 8),
    (2, 8, 2, 1, 6, 640, [600, 31], 2),
    (1, 16, 3, 1, 4, 256, [200], 30),                   # peaked: one key has nearly all
    (2, 33, 4, 1, 5, 448, [448, 5], 2),
    (1, 64, 4, 2, 6, 704, [650], 2),
    (1, 64, 1, 1, 16, 128, [100], 4),
    (4, 3, 1, 1, 1, 2176, [2100, 0, 9999, -7], 2),      # lengths past the cache and below zero are clamped
]


@pytest.mark.gpu
@pytest.mark.parametrize("kv_splits", [0, 1, 3])
@pytest.mark.parametrize("B,T,kids,H,ratio,cap,lens,sharp", ATTENTIONS)
def test_attention_tree(rt4, torch_gpu, orc, B, T, kids, H, ratio, cap, lens, sharp, kv_splits):
    print(f"case attention B={B} T={T} H={H} ratio={ratio} cap={cap} lens={lens} splits={kv_splits}", flush=True)
    rng = np.random.default_rng(B * 100 + T)
    TP = B * T + 3
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, cap, sharp, TP)
    parent = np.array([random_tree(rng, T, kids) for _ in range(B)])
    spoil_unseen(kv, draft, lens, T)
    out = torch_gpu.full((H * ratio, TP, D), 7.0, device="cuda")
    rt4.attention_tree(dev(qq), dev(qs), *map(dev, kv), dev(np.array(lens)), *map(dev, draft), dev(parent), ratio=ratio,
                       kv_max=min(cap, max(0, max(lens))), out=out, kv_splits=kv_splits)
    check_attention(out, *tree_attention(qq, qs, kv, lens, draft, parent, ratio))
    assert (host(out)[:, B * T:] == 7.0).all()          # rows behind the last node


@pytest.mark.gpu
def test_attention_padding_idle_and_no_cache(rt4, torch_gpu, orc):
    """Padding nodes, broken chains and idle sequences give zeros, whatever their K/V; a cache is optional."""
    rng = np.random.default_rng(3)
    B, T, H, ratio = 4, 7, 2, 3
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, 128, 2)
    parent = np.array([[-1, 0, 1, 1, -1, 4, 9], [-2, 0, 1, 2, 3, 4, 5], [-1, -1, -1, -1, -1, -1, -1], [-1, 0, 0, 3, 2, 5, -7]])
    for x in (1, 3):
        draft[x][1] = np.nan                            # the idle sequence's tile was never written
    lens = [70, 128, 0, 1]
    for cache in (kv, None):
        out = rt4.attention_tree(dev(qq), dev(qs), *(map(dev, cache) if cache else [None] * 4), dev(np.array(lens)) if cache else None,
                                 *map(dev, draft), dev(parent), ratio=ratio)
        want, tol = tree_attention(qq, qs, cache, lens, draft, parent, ratio)
        check_attention(out, want, tol)
        o = host(out)
        assert (o[:, 4:7] == 0).all() and (o[:, 7:14] == 0).all() and (o[:, 15:21] == 0).all() and (o[:, 24] == 0).all()
        assert (o[:, 0] != 0).any() and (o[:, 14] != 0).any()


@pytest.mark.gpu
def test_attention_lengths_beyond_the_plan(rt4, torch_gpu, orc):
    """kv_max is a hint: longer sequences are right, and every split count gives one answer up to rounding."""
    rng = np.random.default_rng(8)
    qq, qs, kv, draft = attention_case(orc, rng, 2, 4, 1, 6, 1408, 2)
    parent = np.array([[-1, 0, 1, 2], [-1, 0, 0, 1]])
    lens = [1400, 700]
    want, tol = tree_attention(qq, qs, kv, lens, draft, parent, 6)
    for kv_max in (0, 64, 1400):
        for splits in (0, 2, 5, 64, 65, 128):
            out = rt4.attention_tree(dev(qq), dev(qs), *map(dev, kv), dev(np.array(lens)), *map(dev, draft), dev(parent), ratio=6,
                                     kv_max=kv_max, kv_splits=splits)
            check_attention(out, want, tol)


def check_verify(rt4, logits, draft, parent, u, temp, q=None, kids=None, kv_len=None, pad=0):
    import torch
    want = verify(logits, draft, parent, u, temp, q, kids)
    lg = dev(np.pad(logits, ((0, 0), (0, pad)), constant_values=1e9))[:, :logits.shape[1]]      # rows may be strided
    qd = None if q is None else dev(np.pad(q, ((0, 0), (0, pad)), constant_values=1.0))[:, :q.shape[1]]
    n0 = None if kv_len is None else dev(np.array(kv_len))
    got = rt4.verify_tree(lg, dev(draft), dev(parent), dev(u), temp=dev(np.array(temp, np.float32)), draft_probs=qd, max_children=kids,
                          kv_len=n0)
    torch.cuda.synchronize()
    for name, g, w in zip(("tokens", "path", "count"), got, want):
        assert np.array_equal(host(g), w), (name, host(g), w)
    if kv_len is not None:
        assert np.array_equal(host(n0), np.array(kv_len) + want[2])
    return want


def verify_case(rng, B, T, V, kids, probs, noise=0.5):
    logits = (rng.standard_normal((B * T, V)) * 2.5).astype(np.float32)
    parent = np.array([random_tree(rng, T, kids) for _ in range(B)])
    at = np.arange(B)[:, None] * T + np.maximum(parent, 0)
    seen = logits + noise * rng.standard_normal(logits.shape)
    draft, q = np.zeros((B, T), np.int64), None
    if probs:
        q = np.exp(seen - seen.max(-1, keepdims=True))
        q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
        for b in range(B):
            for i in range(T):
                w = q[at[b, i]].astype(np.float64)
                draft[b, i] = rng.choice(V, p=w / w.sum())
    else:
        for b in range(B):
            for i in range(1, T):
                rank = list(parent[b, 1:i]).count(parent[b, i])
                draft[b, i] = np.argsort(-seen[at[b, i]])[min(rank, V - 1)]
    return logits, draft, parent, rng.random((B, T)).astype(np.float32), q


VERIFIES = [(1, 1, 1), (1, 1, 2), (1, 1, 4097), (2, 4, 63), (1, 4, 70001), (3, 9, 4096), (2, 64, 300), (5, 16, 12289), (1, 2, 1 << 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,T,V", VERIFIES)
def test_verify_tree(rt4, torch_gpu, B, T, V, probs):
    rng = np.random.default_rng(B * 77 + T + V)
    for kids in sorted({1, 2, 3} if T > 1 else {1}):
        print(f"case verify B={B} T={T} V={V} kids={kids} probs={probs}", flush=True)
        logits, draft, parent, u, q = verify_case(rng, B, T, V, kids, probs)
        temp = [(1.0, 0.7, 0.0, 3.0, -1.0)[b % 5] for b in range(B)]
        check_verify(rt4, logits, draft, parent, u, temp, q, kids if probs else None, kv_len=[5] * B, pad=3 * (V < 10000))


@pytest.mark.gpu
def test_verify_accepts_and_rejects_everything(rt4, torch_gpu):
    """Uniforms at both ends: 0 accepts whatever has a probability, 1 - 2^-24 little."""
    rng = np.random.default_rng(9)
    for kids, probs in ((1, False), (3, False), (1, True), (3, True)):
        logits, draft, parent, u, q = verify_case(rng, 2, 12, 1000, kids, probs, noise=0.0)
        for v in (0.0, 1 - 2.0**-24):
            want = check_verify(rt4, logits, draft, parent, np.full_like(u, v), [1.0, 0.5], q, kids if probs else None)
            if v == 0:
                assert (want[2] > 1).all()


@pytest.mark.gpu
def test_verify_odd_rows(rt4, torch_gpu):
    """Masked, infinite and NaN logits, ties, empty rows, tokens outside the vocabulary, repeated siblings, idle and broken trees."""
    rng = np.random.default_rng(11)
    T, V = 6, 9000
    parent = np.array([[-1, 0, 0, 0, 1, 2]] * 7 + [[-3, 0, 1, 2, 3, 4], [-1, -1, 1, 0, 9, 3]])
    B = len(parent)
    logits = rng.standard_normal((B, T, V)).astype(np.float32)
    draft = rng.integers(0, V, (B, T))
    logits[0, :, 100:] = -np.inf                        # a grammar that leaves few tokens
    draft[0] = [0, 5, 200, 7, 3, 4]
    logits[1, :, 7] = np.nan
    logits[1, :, 8] = np.inf                            # all the mass on one token, or on two
    logits[1, :, 4500] = np.inf
    draft[1] = [0, 7, 8, 4500, 8, 8]
    logits[2] = -np.inf                                 # nothing can be drawn
    draft[3] = [0, -1, V, 2**31 - 1, 5, 5]              # no such tokens
    logits[4, :, 3000:3010] = 50.0                      # ties of the largest
    draft[4] = [0, 3001, 3000, 3002, 3000, 3000]
    draft[5] = [0, 77, 77, 77, 1, 1]                    # the same token three times
    logits[5, 0, 77] = 9.0
    logits[6] = np.finfo(np.float32).min                # a mask of the type's lowest value, over a whole row and in part
    logits[6, 0, 10:20] = 1.0
    draft[6] = [0, 12, 13, 14, 12, 12]
    flat = logits.reshape(B * T, V)
    q = np.full((B * T, V), 1.0 / V, np.float32)
    for temp in ([1.0] * B, [0.0] * B, [float("nan")] * B, [1e-3] * B, [1e3] * B):
        for rep in range(4):
            u = rng.random((B, T)).astype(np.float32)
            check_verify(rt4, flat, draft, parent, u, temp)
            check_verify(rt4, flat, draft, parent, u, temp, q, 1)
            if temp[0] != 1e-3:                         # (equal mass on few tokens and a tiny residual: still exact)
                check_verify(rt4, flat, draft, parent, u, temp, q, 3)


# ------------------------------------------------------------ as one would use them --
def decode_steps(rt4, torch, seed, steps, B=2, T=6, H=2, ratio=3, cap=256, V=2000, graph=False):
    """A few verify steps: draft tile, attention, logits from it, verification, append of the accepted path."""
    rng = np.random.default_rng(seed)
    QH = H * ratio
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    zi = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = [zi(B, H, cap, 32), z(B, H, 2, cap), zi(B, H, cap // 8, D), z(B, H, cap // BG, D)]
    stage, draft = z(B, H, BG, D), [zi(B, H, BG, 32), z(B, H, 2, BG), zi(B, H, 8, D), z(B, H, 1, D)]
    kv_len = zi(B)
    # prompts of two lengths
    n0 = np.array([70, 3])
    kf, vf = (dev(rng.standard_normal((B, 70, H, D)).astype(np.float32)) for _ in range(2))
    kv_len.copy_(dev(n0))
    rt4.kv_append_rows(*kv, stage, kf, vf, kv_len=kv_len, count=dev(n0))
    q, kf, vf, toks, par, u = z(B * T, QH, D), z(B, T, H, D), z(B, T, H, D), zi(B, T), zi(B, T), z(B, T)
    wq = dev(rng.integers(0, 2**32, (V, QH * D // 8), dtype=np.uint32))
    wsc = dev((rng.random((QH * D // G, V)) * 0.05).astype(np.float32))
    tokens, path, count = zi(B, T), zi(B, T), zi(B)
    out, logits = z(QH, B * T, D), z(B * T, V)
    qq, qs = zi(QH, B * T, 32), z(QH, 2, B * T)

    def step():
        rt4.attn_q_quant(q, B * T, qq=qq, qs=qs)
        rt4.kv_append_rows(*draft, None, kf, vf)
        rt4.attention_tree(qq, qs, *kv, kv_len, *draft, par, ratio=ratio, out=out)
        rt4.gemm_w4a8_i8(wq, wsc, *rt4.quant_rows_i8(out.permute(1, 0, 2).reshape(B * T, QH * D)), out=logits)
        rt4.verify_tree(logits, toks, par, u, kv_len=kv_len, tokens=tokens, path=path, count=count)
        rt4.kv_append_rows(*kv, stage, kf, vf, kv_len=kv_len, rows=path, count=count)

    g = None
    seen = []
    for s in range(steps):
        q.copy_(dev((rng.standard_normal((B * T, QH, D)) / 8).astype(np.float32)))
        kf.copy_(dev(rng.standard_normal((B, T, H, D)).astype(np.float32)))
        vf.copy_(dev(rng.standard_normal((B, T, H, D)).astype(np.float32)))
        par.copy_(dev(np.array([random_tree(rng, T, 2) for _ in range(B)])))
        toks.copy_(dev(rng.integers(0, 4, (B, T))))
        u.copy_(dev((rng.random((B, T)) * 0.002).astype(np.float32)))     # (small: random drafts are accepted now and then)
        if graph and s == 1:
            torch.cuda.synchronize()
            keep = kv_len.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
            assert torch.equal(kv_len, keep)            # (captured, not run)
        if g is not None:
            g.replay()
        else:
            step()
        torch.cuda.synchronize()
        seen.append([host(x).copy() for x in (out, logits, tokens, path, count, kv_len, kf, vf)])
    return seen, [host(x) for x in (*kv, stage)], n0, [host(x) for x in (qq, qs, *draft, par, toks, u)]


@pytest.mark.gpu
def test_decode_steps(rt4, torch_gpu, orc):
    """Several steps: lengths, the caches' valid keys and stages equal the oracle's appends of the accepted rows."""
    print("case decode steps", flush=True)
    seen, kv, n0, _ = decode_steps(rt4, torch_gpu, 4, 12)
    B, T, H = seen[0][6].shape[:3]
    cap = kv[0].shape[2]
    rng = np.random.default_rng(4)
    kf, vf = (rng.standard_normal((B, 70, H, D)).astype(np.float32) for _ in range(2))
    want = [np.zeros((B, H, cap, 32), np.uint32), np.zeros((B, H, 2, cap), np.float32), np.zeros((B, H, cap // 8, D), np.uint32),
            np.zeros((B, H, cap // BG, D), np.float32)]
    stage = np.zeros((B, H, BG, D), np.float32)
    append_expected(orc, want, stage, kf, vf, np.zeros(B, int), np.tile(np.arange(70), (B, 1)), n0)
    length = n0.copy()
    total = 0
    for out, logits, tokens, path, count, kv_len, kf, vf in seen:
        assert np.isfinite(out).all()
        append_expected(orc, want, stage, kf, vf, length, path, count)
        length = length + count
        total += int((count > 1).sum())
        assert np.array_equal(kv_len, length)
        for b in range(B):
            n = count[b]
            assert (path[b, :n] >= 0).all() and (path[b, n:] == -1).all() and (tokens[b, :n] >= 0).all() and (tokens[b, n:] == -1).all()
    assert total > 0                                    # some drafts were accepted
    for name, g, w in zip(("kc", "ksc", "vc", "vsc", "stage"), kv, (*want, stage)):
        assert np.array_equal(g.view(np.uint32), w.view(np.uint32)), name


@pytest.mark.gpu
def test_decode_steps_captured(rt4, torch_gpu):
    """A step captured once and replayed for every later token gives the eager steps' bits, lengths advancing on the device."""
    print("case decode steps, captured", flush=True)
    eager, kv, _, _ = decode_steps(rt4, torch_gpu, 6, 8)
    again, kv2, _, _ = decode_steps(rt4, torch_gpu, 6, 8, graph=True)
    for a, b in zip(eager, again):
        for x, y in zip(a, b):
            assert np.array_equal(x, y)
    for x, y in zip(kv, kv2):
        assert np.array_equal(x.view(np.uint32), y.view(np.uint32))


@pytest.mark.gpu
def test_side_stream(rt4, torch_gpu, orc):
    """Calls go to the current stream: behind slow work on a side stream they still see its results."""
    torch = torch_gpu
    rng = np.random.default_rng(2)
    logits, draft, parent, u, _ = verify_case(rng, 2, 5, 5000, 2, False)
    want = verify(logits, draft, parent, u, [1.0, 1.0])
    args = [dev(x) for x in (draft, parent, u)]
    src, lg = dev(logits), torch.zeros(logits.shape, device="cuda")
    big = torch.randn((2048, 2048), device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(20):
            big = big @ big * 1e-3
        lg.copy_(src)
        got = rt4.verify_tree(lg, *args)
    s.synchronize()
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w)


@pytest.mark.gpu
def test_python_refusals_on_the_device(rt4, torch_gpu):
    torch = torch_gpu
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ok = dict(logits=f(4, 10), draft=i(1, 4), parent=i(1, 4), u=f(1, 4))
    rt4.verify_tree(**ok)
    for bad in (dict(logits=f(4, 10).half()), dict(logits=f(5, 10)), dict(logits=f(10, 4).T), dict(draft=i(1, 4).long()),
                dict(u=f(4)), dict(u=torch.zeros(1, 4)), dict(draft_probs=f(4, 10)), dict(max_children=2), dict(temp=f(2)),
                dict(kv_len=i(2)), dict(parent=i(1, 65))):
        with pytest.raises(rt4.RT4Error):
            rt4.verify_tree(**{**ok, **bad})
    kv = lambda cap=64: (i(1, 2, cap, 32), f(1, 2, 2, cap), i(1, 2, cap // 8, D), f(1, 2, cap // 64, D))  # noqa: E731
    x = f(1, 4, 2, D)
    rt4.kv_append_rows(*kv(), None, x, x)
    for bad in (dict(kv_len=i(1)), dict(rows=i(1, 5)), dict(count=i(2)), dict(kf=f(1, 4, 3, D)), dict(stage=f(1, 2, 32, D))):
        with pytest.raises(rt4.RT4Error):
            rt4.kv_append_rows(*kv(), **{**dict(stage=None, kf=x, vf=x), **bad})
    q = (i(4, 4, 32), f(4, 2, 4))
    rt4.attention_tree(*q, *kv(128), i(1), *kv(), i(1, 4), ratio=2)
    for a, k in (((*q, *kv(128), i(1), *kv(128), i(1, 4)), dict(ratio=2)), ((*q, *kv(128), i(1), *kv(), i(1, 5)), dict(ratio=2)),
                 ((*q, *kv(128), i(1), *kv(), i(1, 4)), dict(ratio=3)), ((*q, *kv(128), i(1), *kv(), i(1, 4)), dict(ratio=2, kv_max=129)),
                 ((*q, *kv(128), i(1).long(), *kv(), i(1, 4)), dict(ratio=2))):
        with pytest.raises(rt4.RT4Error):
            rt4.attention_tree(*a, **k)


@pytest.mark.gpu
def test_many_sequences(rt4, torch_gpu, orc):
    """More sequences than a wave has lanes, of all lengths: the shares of the keys, the joins and the walks."""
    rng = np.random.default_rng(21)
    B, T, H, ratio, cap = 150, 2, 1, 2, 192
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, cap, 2)
    lens = rng.integers(-1, cap + 2, B)
    parent = np.tile([[-1, 0]], (B, 1))
    parent[rng.integers(0, B, 20), 0] = -2
    spoil_unseen(kv, draft, lens, T)
    want, tol = tree_attention(qq, qs, kv, lens, draft, parent, ratio)
    for splits in (0, 1, 2, 100):
        print(f"case many sequences, kv_splits={splits}", flush=True)
        out = rt4.attention_tree(dev(qq), dev(qs), *map(dev, kv), dev(lens), *map(dev, draft), dev(parent), ratio=ratio, kv_splits=splits)
        check_attention(out, want, tol)
    for probs in (False, True):
        logits, tok, par, u, q = verify_case(rng, B, 5, 500, 2, probs)
        check_verify(rt4, logits, tok, par, u, [(1.0, 0.0)[b % 2] for b in range(B)], q, 2 if probs else None, kv_len=list(range(B)))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(rt4, torch_gpu, orc):
    """The longest cache there may be, 2^24 - 64 keys, for two sequences: byte offsets pass 2^31 within one and 2^32 over both."""
    torch = torch_gpu
    print("case longest cache", flush=True)
    cap, B, H, ratio, T = (1 << 24) - 64, 2, 1, 2, 2
    g = torch.Generator(device="cuda").manual_seed(7)
    ri = lambda *s: torch.randint(-2**31, 2**31 - 1, s, dtype=torch.int32, device="cuda", generator=g)  # noqa: E731
    kv = [ri(B, H, cap, 32), torch.rand((B, H, 2, cap), device="cuda", generator=g), ri(B, H, cap // 8, D),
          torch.rand((B, H, cap // BG, D), device="cuda", generator=g)]
    rng = np.random.default_rng(7)
    lens = [cap - 70, cap - 3]
    # the last keys, through the append (within a tile, and to the cache's very end)
    kf, vf = (rng.standard_normal((B, 3, H, D)).astype(np.float32) for _ in range(2))
    stage = rng.standard_normal((B, H, BG, D)).astype(np.float32)
    tail = [host(x) for x in (kv[0][:, :, -128:], kv[1][:, :, :, -128:], kv[2][:, :, -16:], kv[3][:, :, -2:])]
    tail = [np.ascontiguousarray(x).view(np.uint32) if x.dtype == np.int32 else np.ascontiguousarray(x) for x in tail]
    st = dev(stage)
    rt4.kv_append_rows(*kv, st, dev(kf), dev(vf), kv_len=dev(np.array(lens) + 3))
    lens = [n + 3 for n in lens]
    append_expected(orc, tail, stage, kf, vf, np.array([128 - 70, 128 - 3]), np.tile(np.arange(3), (B, 1)), np.array([3, 3]))
    for g_, w in zip((kv[0][:, :, -128:], kv[1][:, :, :, -128:], kv[2][:, :, -16:], kv[3][:, :, -2:], st), (*tail, stage)):
        assert np.array_equal(np.ascontiguousarray(host(g_)).view(np.uint32), w.view(np.uint32))
    # attention over all of it, against 64-bit sums by pieces
    qq, qs, _, draft = attention_case(orc, rng, B, T, H, ratio, BG, 0.2)
    parent = np.array([[-1, 0], [-1, 0]])
    out = rt4.attention_tree(dev(qq), dev(qs), *kv, dev(np.array(lens)), *map(dev, draft), dev(parent), ratio=ratio)
    nib = lambda w: torch.stack([(w << (28 - 4 * e)) >> 28 for e in range(8)], -1)  # noqa: E731
    for b in range(B):
        Kd, Vd = cache_values(*(x[b, 0] for x in draft))
        for r in range(ratio):
            for i in range(T):
                q = nibbles(qq[r, b * T + i]).reshape(D) * np.repeat(qs[r, :, b * T + i].astype(np.float64), G)
                s_d = Kd[:i + 1] @ q
                qd = torch.tensor(q, device="cuda")
                parts, top, step = [], s_d.max(), 1 << 21
                for k0 in range(0, lens[b], step):
                    k1 = min(k0 + step, lens[b])
                    kk = nib(kv[0][b, 0, k0:k1]).reshape(k1 - k0, D).double()
                    s = (kk[:, :G] @ qd[:G]) * kv[1][b, 0, 0, k0:k1].double() + (kk[:, G:] @ qd[G:]) * kv[1][b, 0, 1, k0:k1].double()
                    del kk
                    m = float(s.max())
                    p = (s - m).exp()
                    t0, t1 = k0 // BG, (k1 + BG - 1) // BG
                    pt = torch.zeros((t1 - t0) * BG, dtype=torch.float64, device="cuda")
                    pt[:k1 - k0] = p
                    v = nib(kv[2][b, 0, t0 * 8:t1 * 8]).transpose(1, 2).reshape(-1, BG, D).float()
                    o = (torch.bmm(pt.view(-1, 1, BG).float(), v)[:, 0].double() * kv[3][b, 0, t0:t1].double()).sum(0)
                    parts.append((m, float(p.sum()), host(o)))
                    top = max(top, m)
                pd = np.exp(s_d - top)
                l = pd.sum() + sum(ls * np.exp(m - top) for m, ls, _ in parts)
                o = pd @ Vd[:i + 1] + sum(o * np.exp(m - top) for m, _, o in parts)
                got = host(out)[r, b * T + i].astype(np.float64)
                # as in tree_attention with |V| <= 8, S <= 2 x 16 x 16 x 0.2 x .. below 64, and the pieces' own fp32 products
                bound = 8 * ((8 * 64 + 168 + 128) * 2.0**-24 + 2.0**-22 + lens[b] * 2.0**-32)
                assert np.abs(got - o / l).max() <= bound, (np.abs(got - o / l).max(), bound)


CAPTURE = r"""
import sys
sys.path[:0] = [{root!r}, {pkg!r}]
import torch
import rt4_amd
torch.cuda.set_device(0)
g = torch.Generator(device="cuda").manual_seed(3)
f = lambda *s: torch.randn(s, device="cuda", generator=g)
i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
B, T, H, ratio, cap, V = 2, 4, 2, 3, 4096, 30000
kv = (i(B, H, cap, 32), torch.ones((B, H, 2, cap), device="cuda"), i(B, H, cap // 8, 256), torch.ones((B, H, cap // 64, 256), device="cuda"))
dr = (i(B, H, 64, 32), torch.ones((B, H, 2, 64), device="cuda"), i(B, H, 8, 256), torch.ones((B, H, 1, 256), device="cuda"))
stage = torch.zeros((B, H, 64, 256), device="cuda")
kv_len = torch.tensor([4000, 77], dtype=torch.int32, device="cuda")
for k in range(0, 4096, 512):
    n = torch.full((B,), k + 512, dtype=torch.int32, device="cuda")
    rt4_amd.kv_append_rows(*kv, stage, f(B, 512, H, 256), f(B, 512, H, 256), kv_len=n)
kf, vf = f(B, T, H, 256), f(B, T, H, 256)
qq, qs = rt4_amd.attn_q_quant(f(B * T, H * ratio, 256) / 8, B * T)
parent = torch.tensor([[-1, 0, 0, 1], [-1, 0, 1, 2]], dtype=torch.int32, device="cuda")
logits, u = f(B * T, V), torch.rand((B, T), device="cuda", generator=g)
draft = logits.view(B, T, V)[:, :1].topk(T, -1).indices[:, 0].int().contiguous()
out = torch.empty((H * ratio, B * T, 256), device="cuda")
outs = (i(B, T), i(B, T), i(B))

def attention(o=None):
    rt4_amd.kv_append_rows(*dr, None, kf, vf)
    return rt4_amd.attention_tree(qq, qs, *kv, kv_len, *dr, parent, ratio=ratio, out=o)

def verify(o=(None, None, None)):
    return rt4_amd.verify_tree(logits, draft, parent, u, tokens=o[0], path=o[1], count=o[2])

def capture(fn):
    gr, err = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(gr):
        try:
            fn()
        except rt4_amd.RT4Error as e:
            err = str(e)
    return gr, err

torch.cuda.synchronize()
ga, err = capture(lambda: attention(out))
print("attention, first call:", err, flush=True)
assert err is None                                        # one unit a sequence needs no workspace
_, err = capture(lambda: verify(outs))
print("verification, first call:", err, flush=True)
assert err is not None and "captur" in err
want, wv = attention().clone(), [x.clone() for x in verify()]
gv, err = capture(lambda: verify(outs))
assert err is None, err
gb, err = capture(lambda: attention(out))
assert err is None, err
for rep in range(3):
    for gr in (ga, gb):
        out.fill_(7.0)
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        rel = float((out - want).norm() / want.norm())
        assert rel < 2 * 168 * 2.0**-24 and (gr is ga or torch.equal(out, want)), rel        # (sums in another order)
    for x in outs:
        x.fill_(9)
    attention()                                           # the program's own work between the replays
    gv.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, wv))
rt4_amd.release_scratch()
again = attention()
assert torch.equal(again, want) and all(torch.equal(a, b) for a, b in zip(verify(), wv))
print("CAPTURE-OK", flush=True)
"""


@pytest.mark.gpu
def test_capture_before_any_eager_call():
    """In a fresh process nothing is allocated under capture: the attention takes one unit a sequence, the verification refuses."""
    import subprocess
    import sys

    from conftest import PKG_DIR, ROOT
    print("case capture in a fresh process", flush=True)
    r = subprocess.run([sys.executable, "-u", "-c", CAPTURE.format(root=str(ROOT), pkg=str(PKG_DIR))], capture_output=True, text=True,
                       timeout=300)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and "CAPTURE-OK" in r.stdout


@pytest.mark.gpu
def test_verify_rejected_mass_leaves_nothing(rt4, torch_gpu):
    """A run of the vocabulary whose only tokens were rejected has no mass: u = 0 draws the first token with any behind it."""
    print("case rejected mass", flush=True)
    rng = np.random.default_rng(11)
    B, T, V = 64, 3, 9000
    logits = np.full((B * T, V), -np.inf, np.float32)
    first = logits[::T]
    first[:, 3], first[:, 5], first[:, 8000] = 0.0, -rng.random(B) - 0.1, -rng.random(B)
    draft, parent = np.tile([0, 3, 5], (B, 1)), np.tile([-1, 0, 0], (B, 1))
    u = np.tile(np.array([0.0, 1 - 2.0**-23, 1 - 2.0**-23], np.float32), (B, 1))
    want = verify(logits, draft, parent, u, np.ones(B))
    assert (want[0][:, 0] == 8000).all() and (want[2] == 1).all()
    got = rt4.verify_tree(dev(logits), dev(draft), dev(parent), dev(u))
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w)


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [False, True])
def test_verify_infinite_temperature(rt4, torch_gpu, probs):
    """At an infinite temperature every token whose logit is not -inf weighs the same."""
    print(f"case infinite temperature probs={probs}", flush=True)
    rng = np.random.default_rng(12)
    B, T, V = 8, 4, 6000
    logits = rng.standard_normal((B * T, V)).astype(np.float32)
    parent = np.tile([-1, 0, 0, 1], (B, 1))
    draft = rng.integers(0, V, (B, T))
    # uniforms between the multiples of 1 / V, so that no sum's rounding decides
    u = ((rng.integers(0, V, (B, T)) + 0.5) / V).astype(np.float32)
    u[::2, 1:] = 0.25 / V
    q = None
    if probs:
        q = rng.random((B * T, V)).astype(np.float32)
        q /= q.sum(1, keepdims=True)
        q[np.arange(B) * T, draft[:, 1]] = 0.5
    temp = np.full(B, np.inf, np.float32)
    want = verify(logits, draft, parent, u, temp, q, 2 if probs else None)
    got = rt4.verify_tree(dev(logits), dev(draft), dev(parent), dev(u), temp=dev(temp), draft_probs=None if q is None else dev(q),
                          max_children=2 if probs else None)
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 7, 63, 64, 65])
def test_shares_of_ragged_lengths(rt4, torch_gpu, orc, B):
    """Planned for any longest length, the keys of sequences of unlike lengths are all shared out."""
    rng = np.random.default_rng(B)
    T, H, ratio, cap = 2, 1, 2, 1024
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, cap, 2)
    lens = np.where(rng.random(B) < 0.3, rng.integers(0, 130, B), rng.integers(0, cap + 1, B))
    lens[-1] = cap
    parent = np.tile([[-1, 0]], (B, 1))
    spoil_unseen(kv, draft, lens, T)
    want, tol = tree_attention(qq, qs, kv, lens, draft, parent, ratio)
    args = [dev(qq), dev(qs), *map(dev, kv), dev(lens), *map(dev, draft), dev(parent)]
    for kv_max in (0, 64, 200, 256, 700, cap):
        print(f"case ragged shares B={B} kv_max={kv_max}", flush=True)
        check_attention(rt4.attention_tree(*args, ratio=ratio, kv_max=kv_max), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("probs,temp,scale", [(False, 1.0, 1.0), (False, 0.0, 1.0), (True, 1.0, 1.0), (False, 1.0, 0.05), (True, 1.0, 0.05)])
def test_verify_star(rt4, torch_gpu, probs, temp, scale):
    """63 children of one root, tokens named twice among them: long runs of rejections, and acceptances late in them."""
    print(f"case star probs={probs} temp={temp} scale={scale}", flush=True)
    rng = np.random.default_rng(31)
    B, T, V = 12, 64, 200
    logits = (rng.standard_normal((B * T, V)) * 2).astype(np.float32)
    parent = np.tile(np.array([-1] + [0] * (T - 1)), (B, 1))
    draft = rng.integers(0, V, (B, T))
    draft[:, 40:] = draft[:, :24]
    u = np.sqrt(rng.random((B, T))).astype(np.float32)
    u[:4, 1:60] = 0.999
    u[:, 1:] *= np.float32(scale)
    q = None
    if probs:
        q = rng.random((B * T, V)).astype(np.float32) ** 4
        q /= q.sum(1, keepdims=True)
    check_verify(rt4, logits, draft, parent, u, [temp] * B, q, T - 1 if probs else None)


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1024), (3, 1, 1025), (2, 1, 32768), (2, 1, 32769), (20, 4, 2047), (5, 10, 1000), (2, 16, 1024), (2, 17, 1024),
                                   (1, 33, 64)])
def test_verify_few_logits(rt4, torch_gpu, B, T, V, probs):
    """Sizes around those that are verified in one launch, chains and drafts that are drawn, greedy and not."""
    print(f"case few logits B={B} T={T} V={V} probs={probs}", flush=True)
    rng = np.random.default_rng(B * 1000 + T + V)
    for kids in (1, 3):
        logits, draft, parent, u, q = verify_case(rng, B, T, V, kids, probs)
        logits[:, ::7] = -np.inf
        if T > 2:
            parent[-1, 0] = -3                          # an idle sequence
        temp = [(1.0, 0.0, 0.3)[b % 3] for b in range(B)]
        check_verify(rt4, logits, draft, parent, u, temp, q, 1 if probs else None, kv_len=list(range(B)), pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,V", [(40, 3, 20000), (2, 4, 1 << 20), (300, 2, 9001)])
def test_verify_repeats(rt4, torch_gpu, B, T, V):
    """The workgroup that draws is whichever ends last: the same tokens every time, from calls right behind one another too."""
    print(f"case repeats B={B} T={T} V={V}", flush=True)
    torch = torch_gpu
    g = torch.Generator(device="cuda").manual_seed(B)
    logits = 2.5 * torch.randn((B * T, V), device="cuda", generator=g)
    q = torch.softmax(logits + 0.5 * torch.randn((B * T, V), device="cuda", generator=g), -1)
    draft = torch.randint(0, V, (B, T), dtype=torch.int32, device="cuda", generator=g)
    draft[:, 1] = q.view(B, T, V)[:, 0].argmax(-1).int()
    parent = torch.tensor([list(range(-1, T - 1))] * B, dtype=torch.int32, device="cuda")
    u = torch.rand((B, T), device="cuda", generator=g)
    outs = [[torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((B, T), (B, T), (B,))] for _ in range(12)]
    for o in outs:
        rt4.verify_tree(logits, draft, parent, u, draft_probs=q, max_children=1, tokens=o[0], path=o[1], count=o[2])
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))
    n = 8 if V < 100000 else 2                          # the first sequences against the walk in 64 bits
    h = [host(x) for x in (logits[:n * T], draft[:n], parent[:n], u[:n], q[:n * T])]
    want = verify(h[0], h[1], h[2], h[3], [1.0] * n, h[4], 1)
    for a, b in zip(outs[0], want):
        assert np.array_equal(host(a)[:n], b)
