"""Edges of the 8-bit linears, gated halves and norms between blocks: values that are not finite, work memory that calls share,
rows of one element."""
from __future__ import annotations

import math

import pytest

from test_ffn import codes8, near, natural, product, rms64, right_codes, U


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("out", ["act", "rows"])
def test_groups_beside_one_that_is_not_finite(rt4, torch_gpu, out, bad):
    """n = h w / rms(h): an infinite value makes its own group NaN and all others 0 (codes 0, scale 1), a NaN all of them NaN."""
    torch = torch_gpu
    g = torch.Generator().manual_seed(5)
    M, K = 3, 512
    h, w = torch.randn((M, K), generator=g), 1 + 0.1 * torch.randn((K,), generator=g)
    h[1, 200] = bad
    _, (q, s) = rt4.block_norm(h.cuda(), weight=w.cuda(), out=out)
    s = (s.T if out == "rows" else s).cpu()
    want = torch.tensor([1.0, math.nan, 1.0, 1.0]) if math.isinf(bad) else torch.full((4,), math.nan)
    assert not bool(q[1].any())
    assert torch.equal(s[1].isnan(), want.isnan()) and torch.equal(s[1].nan_to_num(7.0), want.nan_to_num(7.0))
    keep = [0, 2]
    codes, _ = right_codes((h[keep].double() * w.double()).reshape(2, 4, 128), 127 if out == "act" else 119)
    assert (natural(q)[keep] == codes.reshape(2, K)).all() and bool((s[keep] > 0).all())


@pytest.mark.gpu
def test_rows_of_one_element(rt4, torch_gpu):
    """The stride of a dimension of one element says nothing: a transposed row is a matrix with rows of one."""
    torch = torch_gpu
    M = 5
    col = lambda dt=torch.float32: torch.arange(1, M + 1, dtype=dt, device="cuda")[None].t()  # noqa: E731  [M, 1], strides (1, M)
    assert col().stride() == (1, M) and col().is_contiguous()
    q, s = rt4.quant_token_a8(col())
    assert torch.equal(q, torch.full_like(q, 127)) and torch.equal(s, col().reshape(M) / 127)
    one = torch.ones(1, device="cuda")
    h = col()
    gate = torch.full((1,), 2.0, device="cuda").as_strided((1,), (7,))
    got, n = rt4.block_norm(h, col(), weight=one, gate=col(), h_out=h, eps=0.0)
    assert got is h and torch.equal(h, col() + col() * col()) and torch.equal(n, torch.ones_like(n))
    got, _ = rt4.block_norm(col(), col(), gate=gate)
    assert torch.equal(got, col() * 3)
    x, sx = codes8(torch, M, 32, 1)
    w, sw = codes8(torch, 1, 32, 2)
    for dtype in (torch.float32, torch.bfloat16):
        out = col(dtype)
        assert rt4.gemm_w8a8(w.cuda(), sw.cuda(), x.cuda(), sx.cuda(), out=out) is out
        near(torch, out, product(torch, x, sx, w, sw), 3 * U, dtype)
    with pytest.raises(rt4.RT4Error):            # rows of two, strided
        rt4.quant_token_a8(torch.ones(2, M, device="cuda").t())


# Products whose K is split, so that their runs' sums meet in memory that a call is given, and one that takes two launches of which
# the second is split: (M, N, K, weights).
SPLIT = [(40, 130, 8208, 1), (40, 130, 8208, 2), (300, 140, 12304, 1), (300, 140, 12304, 2), (13, 21740, 7680, 2)]


@pytest.mark.parametrize("M,N,K,weights", SPLIT)
def test_sizes_that_share_work_memory_are_split(rt4, M, N, K, weights):
    for m in (M, M + 1):
        plan = rt4.w8a8_launch_plan(m, N, K, weights, cus=256)
        assert plan[-1]["splits"] > 1
        assert len(plan) == (2 if N > 1000 else 1)


def split_case(torch, M, N, K, weights, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = lambda r: torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8, device="cuda")  # noqa: E731
    scale = lambda r: torch.rand((r,), generator=g, device="cuda") * 0.01 / math.sqrt(K) + 1e-6  # noqa: E731
    return [(code(N), scale(N)) for _ in range(weights)], code(M), scale(M)


def split_call(rt4, w, x, sx):
    return rt4.gemm_w8a8(*w[0], x, sx) if len(w) == 1 else rt4.ffn_gate_w8a8(*w[0], *w[1], x, sx)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,weights", SPLIT)
def test_split_products_on_two_streams(rt4, torch_gpu, M, N, K, weights):
    """Both streams' calls have work memory of their own, and a call's is free for the next on its stream alone."""
    torch = torch_gpu
    assert rt4.w8a8_launch_plan(M, N, K, weights)[-1]["splits"] > 1
    cases = [split_case(torch, M + i, N, K, weights, i) for i in range(2)]
    want = [split_call(rt4, *c) for c in cases]
    ref = torch.mm(cases[0][1].double(), cases[0][0][0][0].double().t().contiguous())
    if weights == 1:
        near(torch, want[0], ref * cases[0][2].double()[:, None] * cases[0][0][0][1].double(), 3 * U, torch.float32)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(split_call(rt4, *cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,weights", SPLIT)
def test_split_products_captured(rt4, torch_gpu, M, N, K, weights):
    """Two captured graphs of split products, replayed in turn and on two streams at once, among eager calls of the same sizes."""
    torch = torch_gpu
    assert rt4.w8a8_launch_plan(M, N, K, weights)[-1]["splits"] > 1
    cases = [split_case(torch, M + i, N, K, weights, 10 + i) for i in range(2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        split_call(rt4, *cases[0])
    side.synchronize()
    graphs, got = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = split_call(rt4, *c)
            b = split_call(rt4, *c)              # (a second call takes the work memory after the first)
        graphs.append(graph)
        got.append((a, b))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(4):
        for w, x, sx in cases:
            x.copy_(torch.randint_like(x, -128, 128))
        want = [split_call(rt4, *c) for c in cases]
        torch.cuda.synchronize()
        for i, s in enumerate(streams if r & 1 else [side, side]):
            with torch.cuda.stream(s):
                graphs[i].replay()
        again = split_call(rt4, *cases[0])
        torch.cuda.synchronize()
        assert torch.equal(again, want[0])
        for (a, b), w in zip(got, want):
            assert torch.equal(a, w) and torch.equal(b, w), r


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 1), (2, 7), (5, 63), (4, 1001), (1100, 131), (1030, 8), (2, 8193), (1, 20001), (2, 65535), (3, 5120), (2100, 1200),
                                 (2, 65536)])
def test_residual_sum_alone(rt4, torch_gpu, M, K):
    """h + y with neither norm nor factors: a sum of two fp32 values (bf16 is one), rounded once (a sum in 64 bits rounds to the
    same fp32 value, since 53 >= 2 * 24 + 2)."""
    torch = torch_gpu
    g = torch.Generator().manual_seed(M + K)
    wide = torch.randn((M, K + 13), generator=g).cuda()
    y = torch.randn((M, K + 3), generator=g).bfloat16().cuda()
    for a, b in ((wide[:, 5:5 + K], y[:, 1:K + 1]), (wide[:, :K].contiguous(), y[:, :K].contiguous())):
        r, none = rt4.block_norm(a, b)
        assert none is None and torch.equal(r, a + b.float())
        for dtype in (torch.bfloat16, torch.float16):
            h = a.to(dtype)
            r, _ = rt4.block_norm(h, b)
            assert torch.equal(r, (h.float() + b.float()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_gated_half_of_scales_that_are_not_finite(rt4, torch_gpu, M):
    """Gates and ups of either infinity and NaN: act(inf) = inf, act(-inf) = -inf / inf = NaN."""
    torch = torch_gpu
    N, K = 200, 256
    x, sx = codes8(torch, M, K, 8)
    wg, sg = codes8(torch, N, K, 9)
    wu, su = codes8(torch, N, K, 10)
    x[0, :8] = 0
    sg[3], sg[5], sg[7], su[3], su[11], su[13] = math.inf, math.nan, -math.inf, -math.inf, math.inf, math.nan
    g, u = product(torch, x, sx, wg, sg), product(torch, x, sx, wu, su)
    for act in ("silu", "gelu_tanh"):
        e = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        want = g / (1 + torch.exp(-e)) * u
        h = rt4.ffn_gate_w8a8(wg.cuda(), sg.cuda(), wu.cuda(), su.cuda(), x.cuda(), sx.cuda(), act=act).cpu().double()
        assert bool(want.isinf().any()) and bool(want.isnan().any())
        # (an act(g) that fp32 holds no more is 0, and 0 times an infinite up is NaN)
        lost = (g / (1 + torch.exp(-e))).abs() < 2.0 ** -120
        keep = ~(lost & u.isinf())
        assert torch.equal(h.isnan() & keep, want.isnan() & keep)
        assert torch.equal(h.isposinf() & keep, want.isposinf() & keep) and torch.equal(h.isneginf() & keep, want.isneginf() & keep)


@pytest.mark.gpu
@pytest.mark.parametrize("ht,yt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("M,K", [(4, 256), (4, 99), (2100, 1200)])
def test_residuals_that_are_not_finite(rt4, torch_gpu, M, K, ht, yt):
    """Infinities and NaN in h, y and the gate reach their own element of the residual (with a norm behind the block, their row) and
    no other; sums that the type does not hold are infinite."""
    torch = torch_gpu
    ht, yt = getattr(torch, ht), getattr(torch, yt)
    g = torch.Generator().manual_seed(M + K)
    for post in (False, True):
        for gated in (False, True):
            h, y = torch.randn((M, K), generator=g).to(ht), torch.randn((M, K), generator=g).to(yt)
            gate = (0.5 + torch.rand((M, K), generator=g)).to(yt) if gated else None
            pw = 1 + 0.1 * torch.randn((K,), generator=g) if post else None
            h[0, 3], h[1, 9], h[3, 7] = math.inf, math.nan, torch.finfo(ht).max
            y[0, 3], y[0, 17], y[1, 30], y[2, 5], y[3, 7] = -math.inf, -math.inf, math.inf, math.nan, torch.finfo(yt).max
            if gated:
                gate[3, 11], gate[3, 12], gate[3, 13] = math.inf, 0.0, math.nan
                y[3, 12] = math.inf if not post else 1.0
            dev = lambda t: None if t is None else t.cuda()  # noqa: E731
            got, _ = rt4.block_norm(dev(h), dev(y), post_weight=dev(pw), gate=dev(gate), scale=0.75)
            got = got.cpu()
            v = y.double()
            if post:
                v = v * rms64(torch, v, 1e-6) * pw.double()
            v = v * 0.75
            if gated:
                v = v * gate.double()
            want = h.double() + v
            assert bool(want.isnan().any()) and not bool(want[4:].isnan().any())
            rounded = want.float().to(ht)
            assert torch.equal(got.isnan(), rounded.isnan()), (post, gated)
            assert torch.equal(got.isposinf(), rounded.isposinf()) and torch.equal(got.isneginf(), rounded.isneginf()), (post, gated)
            # the sums are off by 2^-40 of their terms at most (a row's squares in 64 bits), so where that does not reach the next
            # rounding they are the nearest ones
            fine = rounded.isfinite()
            e = (h.double().abs() + v.abs()) * 2.0 ** -40
            near_by = (got == (want - e).float().to(ht)) | (got == (want + e).float().to(ht)) | (got == rounded)
            assert bool(near_by[fine].all()), (post, gated)
