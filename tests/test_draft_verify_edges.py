"""Draft-and-verify decode steps where they can go wrong: outstanding keys, idle sequences, plans, capture, a cache's end.

Expectations are those of test_draft_verify.py (64-bit softmax, a literal walk) or, for plans, the launches that a capture
records.
"""
from __future__ import annotations

import ctypes
import subprocess
import sys

import numpy as np
import pytest

from conftest import PKG_DIR, ROOT
from test_draft_verify import (BG, D, append_expected, attention_case, check_attention, check_verify, dev, host, random_tree,
                               tree_attention, verify, verify_case)

pytestmark = pytest.mark.gpu


class _KernelNode(ctypes.Structure):                    # hipKernelNodeParams
    _fields_ = [("block", ctypes.c_uint32 * 3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p), ("grid", ctypes.c_uint32 * 3),
                ("params", ctypes.c_void_p), ("shared", ctypes.c_uint32)]


def recorded(torch, fn):
    """Grids (workgroups) of the launches that fn() makes, in order, from a capture that is not run."""
    path = next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln)
    hip = ctypes.CDLL(path)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph, n = ctypes.c_void_p(), ctypes.c_size_t()
    with torch.cuda.stream(stream):
        assert hip.hipStreamBeginCapture(ctypes.c_void_p(stream.cuda_stream), 2) == 0
        try:
            fn()
        finally:
            assert hip.hipStreamEndCapture(ctypes.c_void_p(stream.cuda_stream), ctypes.byref(graph)) == 0
    assert hip.hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(graph, nodes, ctypes.byref(n)) == 0
    grids = []
    for node in nodes:
        p = _KernelNode()
        assert hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        grids.append(tuple(p.grid))
    assert hip.hipGraphDestroy(graph) == 0
    return grids


# ---------------------------------------------------------------- attention --
@pytest.mark.parametrize("n", [4096, 32768, 131072, 1 << 20])
def test_outstanding_key(rt4, torch_gpu, n):
    """The cache's first key far above all the others, its value small: what the others weigh together counts.

    Every head has its own distance, 10 to 33 nats.  The bound is relative to the output, whose terms are all positive, and
    counts fp32 roundings as test_draft_verify.tree_attention does (8 S + 168, one a tile of a run, one a run in the join) and
    2^-22 for P: no key may be lost for its small weight."""
    torch = torch_gpu
    print(f"case outstanding key n={n}", flush=True)
    QH = 48
    kv = [torch.zeros((1, 1, n, D // 8), dtype=torch.int32, device="cuda"), torch.ones((1, 1, 2, n), device="cuda"),
          torch.full((1, 1, n // 8, D), 0x77777777, dtype=torch.int32, device="cuda"),
          torch.full((1, 1, n // BG, D), np.float32(1 / 7), device="cuda")]
    draft = [torch.zeros((1, 1, BG, D // 8), dtype=torch.int32, device="cuda"), torch.ones((1, 1, 2, BG), device="cuda"),
             torch.full((1, 1, 8, D), 0x77777777, dtype=torch.int32, device="cuda"),
             torch.full((1, 1, 1, D), np.float32(1 / 7), device="cuda")]
    kv[0][0, 0, 0] = 0x11111111
    kv[3][0, 0, 0] = float(np.float32(0.05 / 7))               # the first tile's values are all small
    qq = torch.full((QH, 1, D // 8), 0x11111111, dtype=torch.int32, device="cuda")
    qs = (np.linspace(10, 33, QH) / D).astype(np.float32)
    parent = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")
    s = qs.astype(np.float64) * D                       # 256 products of 1 x 1
    V, V0 = 7 * float(np.float32(1 / 7)), 7 * float(np.float32(0.05 / 7))
    p = np.exp(-s)
    want = (V0 + p * ((BG - 1) * V0 + (n - BG + 1) * V)) / (1 + n * p)
    for splits in (1, 128, 0):
        out = rt4.attention_tree(qq, dev(np.repeat(qs[:, None, None], 2, 1)), *kv, dev(np.array([n])), *draft, parent, ratio=QH,
                                 kv_splits=splits)
        tiles = n / BG / 128 + 128 if splits == 128 else n / BG
        tol = (8 * s * 1.4427 + 168 + tiles) * 2.0**-24 + 2.0**-22
        err = np.abs(host(out)[:, 0].astype(np.float64) / want[:, None] - 1)
        assert (err <= tol[:, None]).all(), (splits, err.max(), (err / tol[:, None]).max())


@pytest.mark.parametrize("value", [2.0**110, 2.0**-110])
def test_large_and_small_values(rt4, torch_gpu, value):
    """A sum over 131072 equal keys is at most their number times their values: it neither overflows nor loses bits sooner."""
    torch = torch_gpu
    print(f"case values of {value}", flush=True)
    n = 131072
    args, kw = blank_attention(torch, 1, 2, 1, 3, n)
    for x in (args[4], args[9]):
        x.fill_(0x11111111)                             # code 1
    for x in (args[5], args[10]):
        x.fill_(value)
    args[11][:, 1] = 0
    for splits in (1, 0):
        out = rt4.attention_tree(*args, **kw, kv_splits=splits)
        assert float((out / value - 1).abs().max()) <= (168 + n / BG) * 2.0**-24 + 2.0**-22


@pytest.mark.parametrize("n", [0, 1, 300])
def test_scores_far_below_zero(rt4, torch_gpu, n):
    """Scores of -1e32 and less, as keys of 1e30 have them: the least of them takes all the weight."""
    torch = torch_gpu
    print(f"case scores far below zero, n={n}", flush=True)
    args, kw = blank_attention(torch, 1, 2, 1, 3, 320)
    args[0].fill_(-1)                                   # codes -1, scale 1
    args[1].fill_(1.0)
    for x in (args[2], args[7]):
        x.fill_(0x11111111)                             # codes 1
    args[3].copy_(1e30 * (2 + torch.arange(320, device="cuda") / 320))
    args[8].fill_(1e30 if n == 0 else 4e30)
    for x in (args[4], args[9]):
        x.random_(-2**31, 2**31 - 1, generator=torch.Generator(device="cuda").manual_seed(n))
    for x in (args[5], args[10]):
        x.fill_(1.0)
    args[6].fill_(n)
    args[11][:, 1] = 0
    first = args[4] if n else args[9]
    want = ((first[0, 0, 0] << 28) >> 28).float()       # V of key 0, or of the root
    if n == 0:
        args[8][0, 0, :, 1] = 2e30                      # node 1 sees the root above its own key
    for splits in (0, 1, 3):
        out = rt4.attention_tree(*args, **kw, kv_splits=splits)
        assert torch.equal(out, want.expand(3, 2, D)), splits


@pytest.mark.parametrize("B,idle,cap", [(1, 1, 256), (3, 1, 32768), (4, 2, 16384), (70, 30, 2048)])
def test_idle_sequences_take_no_share(rt4, torch_gpu, orc, B, idle, cap):
    """Idle sequences' caches are not attended, however long: the others' bits do not depend on them, and their rows are zeros."""
    print(f"case {idle} idle sequences of {B}", flush=True)
    rng = np.random.default_rng(B)
    T, H, ratio = 4, 1, 6
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, cap, 2)
    parent = np.tile([-1, 0, 1, 1], (B, 1))
    parent[-idle:, 0] = -2
    lens = np.array([cap - 3 * b % 200 for b in range(B)])
    for x in (1, 3):
        kv[x][-idle:], draft[x][-idle:] = np.nan, np.nan
    args = [dev(qq), dev(qs), *map(dev, kv)], [*map(dev, draft), dev(parent)]
    outs = []
    for n in (cap, 0, 77):
        lens[-idle:] = n
        outs.append(rt4.attention_tree(*args[0], dev(lens), *args[1], ratio=ratio))
    check_attention(outs[0], *tree_attention(qq, qs, kv, lens, draft, parent, ratio))
    assert (host(outs[0])[:, (B - idle) * T:] == 0).all()
    for o in outs[1:]:
        assert np.array_equal(host(o).view(np.uint32), host(outs[0]).view(np.uint32))


def blank_attention(torch, B, T, H, ratio, cap):
    """Arguments of a call on zeros: (positional, keywords)."""
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    cache = lambda n: (i(B, H, n, D // 8), f(B, H, 2, n), i(B, H, n // 8, D), f(B, H, n // BG, D))  # noqa: E731
    parent = i(B, T)
    parent[:, 0] = -1
    args = (i(H * ratio, B * T, D // 8), f(H * ratio, 2, B * T), *cache(cap), torch.full((B,), cap, dtype=torch.int32, device="cuda"),
            *cache(BG), parent)
    return args, dict(ratio=ratio, out=f(H * ratio, B * T, D))


def test_more_row_groups_than_an_xcd_takes(rt4, torch_gpu):
    """Many rows of one KV head are split over the XCDs too (the groups of one unit stay on one), and come out right."""
    torch = torch_gpu
    print("case 64 nodes of 64 heads over one KV head", flush=True)
    B, T, H, ratio, cap = 1, 64, 1, 64, 8192
    args, kw = blank_attention(torch, B, T, H, ratio, cap)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (args[0], args[2], args[4], args[7], args[9]):
        x.random_(-2**31, 2**31 - 1, generator=g)
    for x in (args[1], args[3], args[5], args[8], args[10]):
        x.uniform_(0.01, 0.02, generator=g)
    out = rt4.attention_tree(*args, **kw).clone()
    one = rt4.attention_tree(*args, **{**kw, "kv_splits": 1})
    grids = recorded(torch, lambda: rt4.attention_tree(*args, **kw))
    assert len(grids) == 2 and grids[0][0] >= 8 * T * ratio // 48, grids      # split, and joined by a second launch
    # two orders of the same sums: S below 2 x 128 x 64 x 0.02^2 x 1.45 = 9.5, values below 8 x 0.02
    tol = 2 * 8 * 0.02 * ((8 * 9.5 + 168 + cap / BG) * 2.0**-24 + 2.0**-22)
    assert float((out - one).abs().max()) <= tol


@pytest.mark.parametrize("B,T,ratio", [(1, 1, 6), (1, 16, 8), (2, 1, 8)])
def test_plan_has_no_more_units_than_there_are(rt4, torch_gpu, B, T, ratio):
    """A sequence has at most 128 units, and no more are planned: few heads over a long cache launch nothing that ends at once."""
    torch = torch_gpu
    print(f"case one KV head, long cache, B={B} T={T}", flush=True)
    args, kw = blank_attention(torch, B, T, 1, ratio, 131072)
    rt4.attention_tree(*args, **kw)
    grids = recorded(torch, lambda: rt4.attention_tree(*args, **kw))
    assert len(grids) == 2 and grids[0][0] <= 128 * B * -(-T * ratio // 16), grids


def in_a_fresh_process(script):
    """Runs a script that prints OK where it succeeds, with this folder and the package at hand."""
    head = f"import sys\nsys.path[:0] = [{str(ROOT)!r}, {str(PKG_DIR)!r}, {str(ROOT / 'tests')!r}]\n"
    r = subprocess.run([sys.executable, "-u", "-c", head + script], capture_output=True, text=True, timeout=100)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and r.stdout.rstrip().endswith("OK")


SPLITS_THAT_FIT = r"""
import torch
import rt4_amd
from test_draft_verify_edges import blank_attention, recorded
args, kw = blank_attention(torch, 1, 1, 1, 6, 131072)
call = lambda **k: rt4_amd.attention_tree(*args, **kw, **k)
assert len(recorded(torch, call)) == 1                    # no workspace: one unit
for n in (3, 50, 100):
    call(kv_splits=n)                                     # (scratch grows by a half at least: 3, 50 and 100 units)
    grids = recorded(torch, call)
    print(n, grids, flush=True)
    assert len(grids) == 2 and grids[0][0] == (n + 7) // 8 * 8, grids
call()
full = recorded(torch, call)
print(full, flush=True)
assert grids[0][0] < full[0][0] <= 128
print("OK", flush=True)
"""


def test_capture_takes_the_splits_that_fit(torch_gpu):
    """Under capture the attention takes as many units as the workspace of earlier calls holds."""
    print("case splits that fit", flush=True)
    in_a_fresh_process(SPLITS_THAT_FIT)


# ------------------------------------------------------------- verification --
ONE_LAUNCH = r"""
import torch
import rt4_amd
from test_draft_verify_edges import recorded
g = torch.Generator(device="cuda").manual_seed(3)

def case(B, T, V, probs):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    logits = 2.5 * torch.randn((B * T, V), device="cuda", generator=g)
    q = torch.softmax(logits + 0.5 * torch.randn((B * T, V), device="cuda", generator=g), -1) if probs else None
    draft = torch.zeros((B, T), dtype=torch.int32, device="cuda")
    draft[:, 1:] = logits.view(B, T, V)[:, :-1].argmax(-1).int()
    parent = torch.arange(-1, T - 1, dtype=torch.int32, device="cuda").repeat(B, 1)
    u = torch.rand((B, T), device="cuda", generator=g)
    outs = (i(B, T), i(B, T), i(B))
    return outs, lambda: rt4_amd.verify_tree(logits, draft, parent, u, draft_probs=q, max_children=1 if probs else None,
                                             tokens=outs[0], path=outs[1], count=outs[2])

CASES = ((1, 1, 16000, 0, 1), (1, 1, 24000, 0, 2), (1, 1, 32768, 0, 2), (3, 4, 4096, 0, 1), (3, 4, 7000, 0, 2), (2, 1, 12000, 1, 1),
         (2, 1, 16000, 1, 2), (2, 2, 10000, 1, 2), (2, 1, 40000, 0, 2), (2, 4, 8000, 1, 2))    # .., launches of a captured call
made = [case(*c[:4]) for c in CASES]
for c, (outs, call) in zip(CASES[:8], made):              # no scratch: one launch in any case
    print(c, recorded(torch, call), flush=True)
    assert len(recorded(torch, call)) == 1
for c, (outs, call) in zip(CASES, made):
    call()                                                # sizes the scratch, whichever form it takes itself
    w = [x.clone() for x in outs]
    n = len(recorded(torch, call))
    print(c, n, flush=True)
    assert n == c[4]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        call()
    for rep in range(3):
        for x in outs:
            x.fill_(9)
        made[-1][1]()                                     # the program's own eager work between the replays
        torch.cuda.synchronize()
        for x in outs:
            x.fill_(9)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
print("OK", flush=True)
"""


def test_verify_in_one_launch_where_it_is_faster(torch_gpu):
    """A captured call takes the form that is faster on the device where its scratch is there, with equal tokens."""
    print("case one launch or two", flush=True)
    in_a_fresh_process(ONE_LAUNCH)


@pytest.mark.parametrize("V", [3000, 70001])
@pytest.mark.parametrize("probs", [False, True])
def test_infinite_logits_at_an_infinite_temperature(rt4, torch_gpu, probs, V):
    """Every logit that is not -inf or NaN weighs the same, +inf ones too."""
    print(f"case infinite logits, infinite temperature, V={V} probs={probs}", flush=True)
    rng = np.random.default_rng(13)
    B, T = 8, 4
    logits = rng.standard_normal((B * T, V)).astype(np.float32)
    logits[:, ::3] = -np.inf
    logits[:, 1::9] = np.nan
    logits[::2, 200:240] = np.inf                       # (among finite ones)
    parent = np.tile([-1, 0, 0, 1], (B, 1))
    draft = rng.choice(np.flatnonzero(np.arange(V) % 9 == 2), (B, T))
    left = np.count_nonzero(logits[0] > -np.inf)
    # uniforms between the multiples of 1 / left, so that no sum's rounding decides
    u = ((rng.integers(0, left - 2, (B, T)) + 0.5) / left).astype(np.float32)
    u[::2, 1:] = 0.25 / left
    q = None
    if probs:
        q = rng.random((B * T, V)).astype(np.float32)
        q /= q.sum(1, keepdims=True)
        q[np.arange(B) * T, draft[:, 1]] = 0.5
    temp = np.full(B, np.inf, np.float32)
    # (the walk in 64 bits divides by the temperature, so it takes the weights' logarithms at temperature 1)
    want = verify(np.where(logits > -np.inf, np.float32(0), np.float32(-np.inf)), draft, parent, u, np.ones(B), q, 2 if probs else None)
    got = rt4.verify_tree(dev(logits), dev(draft), dev(parent), dev(u), temp=dev(temp), draft_probs=None if q is None else dev(q),
                          max_children=2 if probs else None)
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w)


@pytest.mark.parametrize("temp", [1e-3, 1e-30, 1.0])
def test_siblings_with_draft_probabilities_on_odd_rows(rt4, torch_gpu, temp):
    """Equal mass on few tokens and what a cold temperature leaves of the others: three siblings tested against residuals."""
    print(f"case odd rows, siblings, temp={temp}", flush=True)
    rng = np.random.default_rng(17)
    T, V = 6, 9000
    parent = np.array([[-1, 0, 0, 0, 1, 2]] * 6)
    B = len(parent)
    logits = rng.standard_normal((B, T, V)).astype(np.float32)
    draft = rng.integers(0, V, (B, T))
    logits[0, :, 100:] = -np.inf                        # few tokens left
    draft[0] = [0, 5, 200, 7, 3, 4]
    logits[1, :, 7] = np.nan
    logits[1, :, 8] = logits[1, :, 4500] = np.inf       # all the mass on two
    draft[1] = [0, 7, 8, 4500, 8, 8]
    logits[2, :, 3000:3010] = 50.0                      # ties of the largest
    draft[2] = [0, 3001, 3000, 3002, 3000, 3000]
    draft[3] = [0, 77, 77, 77, 1, 1]                    # the same token three times
    logits[3, 0, 77] = 9.0
    logits[4] = np.finfo(np.float32).min                # the type's lowest value, over a whole row and in part
    logits[4, 0, 10:20] = 1.0
    draft[4] = [0, 12, 13, 14, 12, 12]
    logits[5, :, ::2] = -np.inf
    flat = logits.reshape(B * T, V)
    q = np.full((B * T, V), 1.0 / V, np.float32)
    for rep in range(6):
        check_verify(rt4, flat, draft, parent, rng.random((B, T)).astype(np.float32), [temp] * B, q, 3)


@pytest.mark.parametrize("B,T,V,kids", [(1, 4, 300000, 3), (2, 5, 270001, 4), (1, 7, 1 << 19, 2)])
def test_siblings_with_draft_probabilities_on_long_rows(rt4, torch_gpu, B, T, V, kids):
    """Residual levels of rows of more chunks than a wave has lanes."""
    print(f"case long rows, siblings, B={B} T={T} V={V}", flush=True)
    rng = np.random.default_rng(V)
    logits, draft, _, u, q = verify_case(rng, B, T, V, kids, True)
    parent = np.array([[-1] + [0] * kids + [1] * (T - 1 - kids)] * B)
    u[:, 1:] = 0.5 + u[:, 1:] / 2                       # (rejections are what residuals are for)
    for temp in (1.0, 0.7):
        check_verify(rt4, logits, draft, parent, u, [temp] * B, q, kids)


CAPTURED_RESIDUALS = r"""
import numpy as np
import torch
import rt4_amd
from test_draft_verify import dev, verify, verify_case

def case(seed, B, T, V, probs):
    rng = np.random.default_rng(seed)
    logits, draft, _, u, q = verify_case(rng, B, T, V, 2, True)
    parent = np.array([[-1, 0, 0] + [1] * (T - 3)] * B)
    q = q if probs else None
    want = verify(logits, draft, parent, u, np.ones(B), q, 2 if probs else None)
    ins = [dev(x) for x in (logits, draft, parent, u)]
    qd = dev(q) if probs else None
    outs = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((B, T), (B, T), (B,))]
    def call():
        rt4_amd.verify_tree(*ins, draft_probs=qd, max_children=2 if probs else None, tokens=outs[0], path=outs[1], count=outs[2])
    def check(what):
        torch.cuda.synchronize()
        for x, w in zip(outs, want):
            assert np.array_equal(x.cpu().numpy(), w), what
        for x in outs:
            x.fill_(9)
        torch.cuda.synchronize()
    return call, check

def capture(fn):
    gr, err = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(gr):
        try:
            fn()
        except rt4_amd.RT4Error as e:
            err = str(e)
    return gr, err

call, check = case(1, 3, 5, 20000, True)
plain, check_plain = case(2, 8, 12, 20000, False)
more, check_more = case(3, 20, 4, 9000, True)
many, check_many = case(4, 200, 3, 9000, True)
_, err = capture(call)
assert err is not None and "captur" in err, err
plain()                                                   # the statistics' scratch is there, the counters are not
check_plain("first eager call")
_, err = capture(call)
print("without counters:", err, flush=True)
assert err is not None and "captur" in err, err
call()
check("eager")
gr, err = capture(call)
assert err is None, err
for rep in range(4):
    gr.replay()
    check(("replay", rep))
    call()
    check(("eager between", rep))
    (more, many)[rep % 2]()                               # 20, then 200 counters: the graph keeps those that it was captured with
    (check_more, check_many)[rep % 2](("more sequences", rep))
    plain()
    check_plain(("chosen tokens", rep))
g2, err = capture(many)
assert err is None, err
for rep in range(3):
    g2.replay()
    gr.replay()
    check_many(("replay", rep))
    check(("both graphs", rep))
print("OK", flush=True)
"""


def test_captured_residuals(torch_gpu):
    """The workgroup that draws is the last to count itself in: its counters under capture, between eager calls and grown."""
    print("case captured residuals", flush=True)
    in_a_fresh_process(CAPTURED_RESIDUALS)


# ------------------------------------------------------------ as one would use them --
@pytest.mark.parametrize("bad", [np.inf, np.nan, 1e30])
def test_padding_rows_are_appended_as_zeros(rt4, torch_gpu, orc, bad):
    """Whatever a model gives for padding nodes, rows of -1 keep it out of the draft tile's scales."""
    print(f"case padding rows of {bad}", flush=True)
    rng = np.random.default_rng(23)
    B, T, H, ratio = 3, 7, 2, 3
    qq, qs, kv, draft = attention_case(orc, rng, B, T, H, ratio, 128, 2)
    parent = np.array([[-1, 0, 0, 2, -1, 4, 9], [-1, 0, 1, 2, 3, 4, 5], [-2, 0, 0, 0, 0, 0, 0]])
    real = np.array([[1, 1, 1, 1, 0, 0, 0], [1] * 7, [0] * 7], bool)
    rows = np.where(real, np.arange(T), -1)
    kf, vf = (rng.standard_normal((B, T, H, D)).astype(np.float32) for _ in range(2))
    kf[~real] = vf[~real] = bad
    got = [dev(x) for x in draft]
    rt4.kv_append_rows(*got, None, dev(kf), dev(vf), rows=dev(rows))
    append_expected(orc, draft, None, kf, vf, np.zeros(B, int), rows, np.full(B, T))
    for name, g, w in zip(("kd", "ksd", "vd", "vsd"), got, draft):
        assert np.array_equal(host(g).view(np.uint32), w.view(np.uint32)), name
    lens = [100, 128, 64]
    out = rt4.attention_tree(dev(qq), dev(qs), *map(dev, kv), dev(np.array(lens)), *got, dev(parent), ratio=ratio)
    check_attention(out, *tree_attention(qq, qs, kv, lens, draft, parent, ratio))
    o = host(out).reshape(H * ratio, B, T, D)
    assert (o[:, ~real] == 0).all() and (o[:, real] != 0).any(-1).all()


def test_sequences_retired_at_the_cache_end(rt4, torch_gpu, orc):
    """A sequence without room for a whole path is made idle on the device: nothing is lost, nothing passes the cache's end."""
    torch = torch_gpu
    print("case cache end", flush=True)
    rng = np.random.default_rng(19)
    B, T, H, ratio, cap, V = 3, 6, 1, 2, 128, 500
    kv = [torch.zeros((B, H, cap, D // 8), dtype=torch.int32, device="cuda"), torch.zeros((B, H, 2, cap), device="cuda"),
          torch.zeros((B, H, cap // 8, D), dtype=torch.int32, device="cuda"), torch.zeros((B, H, cap // BG, D), device="cuda")]
    want = [np.ascontiguousarray(host(x)).view(np.uint32) if x.dtype == torch.int32 else host(x).copy() for x in kv]
    draft = [torch.zeros((B, H, BG, D // 8), dtype=torch.int32, device="cuda"), torch.zeros((B, H, 2, BG), device="cuda"),
             torch.zeros((B, H, 8, D), dtype=torch.int32, device="cuda"), torch.zeros((B, H, 1, D), device="cuda")]
    stage, wstage = torch.zeros((B, H, BG, D), device="cuda"), np.zeros((B, H, BG, D), np.float32)
    length = np.array([100, 40, 126])
    kv_len = dev(length)
    kf, vf = (rng.standard_normal((B, cap, H, D)).astype(np.float32) for _ in range(2))
    rt4.kv_append_rows(*kv, stage, dev(kf), dev(vf), kv_len=kv_len, count=kv_len)
    append_expected(orc, want, wstage, kf, vf, np.zeros(B, int), np.tile(np.arange(cap), (B, 1)), length)
    retired = np.zeros(B, int)
    for step in range(60):
        kf, vf = (rng.standard_normal((B, T, H, D)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((B * T, H * ratio, D)).astype(np.float32) / 8
        tree = np.array([random_tree(rng, T, 2) for _ in range(B)])
        tok = rng.integers(0, 8, (B, T))
        logits = rng.standard_normal((B * T, V)).astype(np.float32)
        logits[:, :8] += 5
        u = (rng.random((B, T)) * 0.3).astype(np.float32)
        idle = length + T > cap
        parent = dev(tree)
        parent[:, 0] = torch.where(kv_len + T > cap, -2, parent[:, 0])
        rt4.kv_append_rows(*draft, None, dev(kf), dev(vf))
        qq, qs = rt4.attn_q_quant(dev(q), B * T)
        out = host(rt4.attention_tree(qq, qs, *kv, kv_len, *draft, parent, ratio=ratio)).reshape(H * ratio, B, T, D)
        tokens, path, count = (host(x) for x in rt4.verify_tree(dev(logits), dev(tok), parent, dev(u), kv_len=kv_len))
        rt4.kv_append_rows(*kv, stage, dev(kf), dev(vf), kv_len=kv_len, rows=dev(path), count=dev(count))
        assert (out[:, idle] == 0).all() and np.isfinite(out).all() and (np.abs(out[:, ~idle]).max(-1) > 0).all()
        assert (count[idle] == 0).all() and (tokens[idle] == -1).all() and (count[~idle] > 0).all()
        append_expected(orc, want, wstage, kf, vf, length, path, count)
        length = length + count
        retired = np.where(idle, retired, step + 1)
        assert np.array_equal(host(kv_len), length) and (length <= cap).all()
        if idle.all():
            break
    print("steps until retired", retired, "lengths", length, flush=True)
    assert idle.all() and (length > cap - T).all() and retired[2] == 0 and retired[1] > retired[0] > 0
    for name, g, w in zip(("kc", "ksc", "vc", "vsc", "stage"), (*kv, stage), (*want, wstage)):
        assert np.array_equal(host(g).view(np.uint32), w.view(np.uint32)), name
