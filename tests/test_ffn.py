"""8-bit linears, gated halves of feed-forward blocks, and norms between blocks, against their definitions in 64 bits.

Tolerances count roundings, u = 2^-24 for fp32 and half a step of the output type: a product of sums is converted (u) and scaled
twice (2 u); a gated half adds the activation's (each step written at `gate_bound`).  Norms are computed in 64 bits and rounded
once (through fp32 for 16-bit types), so only that is left.  Codes have one right value.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

DUMMY = ctypes.c_void_p(0x1000)          # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1004)
U = 2.0 ** -24


def half_step(torch, dtype):
    return torch.finfo(dtype).eps / 2


def near(torch, got, ref, rel, dtype, flushed=None):
    """|got - ref| within rel of |ref| and the output's rounding (half a step, or half the smallest subnormal), and `flushed`."""
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    top = torch.finfo(dtype).max
    over = fine & (ref.abs() * (1 + 2 * half_step(torch, dtype)) >= top)
    fine &= ~over
    rel = rel if isinstance(rel, float) else rel.double().cpu()[fine]
    tiny = 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126       # (results below fp32's normal numbers may be flushed)
    bound = ref[fine].abs() * ((1 + rel) * (1 + half_step(torch, dtype)) - 1) + tiny
    if flushed is not None:
        bound = bound + flushed.double().cpu()[fine]
    off = (got[fine] - ref[fine]).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()))


def codes8(torch, rows, K, seed, low=-127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, 128, (rows, K), generator=g, dtype=torch.int8), torch.rand((rows,), generator=g) * 0.01 + 1e-3


def product(torch, x, sx, w, sw):
    return (x.double() @ w.double().T) * sx.double()[:, None] * sw.double()


def act64(torch, x, act):
    return x * torch.sigmoid(x) if act == "silu" else x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))


def gate_bound(torch, g, act):
    """Relative error of act(g) * u.  g and u carry 3 u each.  silu: the exponent E = |x| log2 e by a rounded constant and a product,
    2 u of it, so 2 u |x| of the exponential, whose own is 2 u; 1 + e (u), reciprocal (2 u), two products (2 u); g's error passes
    with the factor |x act'(x) / act(x)| <= 1 + |x|.  gelu_tanh: with Z = |2 z|, E = Z log2 e by a square, a fused sum of two rounded
    constants and a product, 5 u of it; g's error passes with at most 1 + 3 Z."""
    x = g.abs()
    if act == "silu":
        return U * (2 * x + 7 + 3 * (1 + x) + 3)
    z = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    return U * (5 * z + 7 + 3 * (1 + 3 * z) + 3)


def gate_flushed(g, u):
    """Absolute error of act(g) * u where the factor 1 / (1 + e) <= 2^-126 of it lies below fp32's normal numbers, which the
    reciprocal gives as 0 (and so does an exponential that overflows, 1 / (1 + e) < 2^-127): what is lost is at most 2^-126 |g u|."""
    return 2.0 ** -126 * (g * u).abs()


SHAPES = [(1, 1, 16), (1, 33, 48), (2, 64, 112), (3, 100, 256), (4, 129, 144), (5, 31, 2064), (16, 160, 320), (17, 257, 1040), (31, 65, 528),
          (33, 500, 64), (64, 300, 400), (65, 640, 208), (100, 1000, 1120), (128, 128, 128), (129, 385, 656), (200, 77, 5120), (257, 513, 272),
          (300, 1100, 1024), (513, 260, 784), (1030, 520, 192), (6, 66, 4112), (7, 10, 16), (8, 1023, 2064), (9, 20, 20000),
          (40, 130, 8208), (130, 70, 16400), (300, 140, 12304), (1024, 2500, 160), (2, 6, 5120)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(rt4, torch_gpu, M, N, K):
    torch = torch_gpu
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, sx = codes8(torch, M, K, 1)
        w, sw = codes8(torch, N, K, 2)
        got = rt4.gemm_w8a8(w.cuda(), sw.cuda(), x.cuda(), sx.cuda(), dtype=dtype)
        assert got.dtype is dtype
        near(torch, got, product(torch, x, sx, w, sw), 3 * U, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated_half(rt4, torch_gpu, M, N, K, act):
    torch = torch_gpu
    x, sx = codes8(torch, M, K, 3)
    wg, sg = codes8(torch, N, K, 4)
    wu, su = codes8(torch, N, K, 5)
    sg = sg * 40 / math.sqrt(K)                  # gates of a few units and some of tens
    g, u = product(torch, x, sx, wg, sg), product(torch, x, sx, wu, su)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = rt4.ffn_gate_w8a8(wg.cuda(), sg.cuda(), wu.cuda(), su.cuda(), x.cuda(), sx.cuda(), act=act, dtype=dtype)
        near(torch, got, act64(torch, g, act) * u, gate_bound(torch, g, act), dtype, gate_flushed(g, u))


# Sizes that take each tile form, whole and with K split, with one and with two weight matrices, and two launches for one call:
# (M, N, K, weights, the (form, whether K is split) of each launch on 256 CUs).
FORM_SIZES = [(3000, 3500, 1040, 1, [(0, 0)]), (400, 12000, 1040, 2, [(0, 0)]), (3391, 735, 18672, 2, [(0, 1)]), (392, 11815, 6496, 2, [(1, 0)]),
              (1703, 6875, 5744, 1, [(1, 0)]), (6730, 324, 16640, 2, [(1, 1)]), (2000, 5000, 2064, 1, [(2, 0)]), (145, 6349, 14912, 2, [(2, 1)]),
              (513, 9000, 2064, 1, [(3, 0)]), (66, 5295, 22944, 1, [(3, 1)]), (10, 25881, 2736, 2, [(4, 0)]), (11, 8056, 18464, 2, [(4, 1)]),
              (9, 31099, 4384, 1, [(5, 0)]), (10, 8631, 17040, 2, [(5, 1)]), (1000, 3500, 112, 1, [(6, 0)]), (79, 3896, 11936, 2, [(6, 1)]),
              (9, 30, 112, 2, [(7, 0)]), (10, 16, 5824, 1, [(7, 1)]), (9, 30, 1040, 1, [(8, 0)]), (9, 16, 12320, 2, [(8, 1)]),
              (700, 12000, 1040, 1, [(6, 0), (8, 0)]), (700, 12000, 1040, 2, [(0, 0), (8, 0)]), (13, 21740, 7680, 2, [(5, 0), (8, 1)]),
              (347, 27804, 9808, 1, [(3, 0), (3, 1)])]


@pytest.mark.parametrize("M,N,K,weights,forms", FORM_SIZES)
def test_forms_are_reached(rt4, M, N, K, weights, forms):
    plan = rt4.w8a8_launch_plan(M, N, K, weights, cus=256)
    assert [(p["form"], int(p["splits"] > 1)) for p in plan] == forms
    assert sum(p["channels"] for p in plan) == N
    assert all(p["tile_m"] % 32 == 0 and p["tile_n"] % 32 == 0 and p["tile_m"] > 0 for p in plan)
    assert [p["form"] for p in rt4.w8a8_launch_plan(8, N, K, weights, cus=256)] == [9]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,weights,forms", FORM_SIZES)
def test_forms(rt4, torch_gpu, M, N, K, weights, forms):
    """Against 64-bit products on the device (sums of K products of codes are exact in them)."""
    torch = torch_gpu
    g = torch.Generator(device="cuda").manual_seed(M + N)
    code = lambda r: torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8, device="cuda")  # noqa: E731
    scale = lambda r: torch.rand((r,), generator=g, device="cuda") * 0.01 / math.sqrt(K) + 1e-6  # noqa: E731
    x, sx = code(M), scale(M)
    w = [(code(N), scale(N)) for _ in range(weights)]
    ref = [torch.mm(x.double(), c.double().t().contiguous()) * sx.double()[:, None] * s.double() for c, s in w]
    if weights == 1:
        near(torch, rt4.gemm_w8a8(*w[0], x, sx), ref[0], 3 * U, torch.float32)
        near(torch, rt4.gemm_w8a8(*w[0], x, sx, dtype=torch.bfloat16), ref[0], 3 * U, torch.bfloat16)
    else:
        got = rt4.ffn_gate_w8a8(*w[0], *w[1], x, sx)
        near(torch, got, act64(torch, ref[0], "silu") * ref[1], gate_bound(torch, ref[0], "silu"), torch.float32, gate_flushed(*ref))


@pytest.mark.gpu
def test_product_without_workspace(rt4, torch_gpu):
    """The C entry without memory for split sums runs unsplit, with the same result; too little is as none."""
    torch = torch_gpu
    M, N, K = 40, 130, 8208
    x, sx = (t.cuda() for t in codes8(torch, M, K, 21))
    w, sw = (t.cuda() for t in codes8(torch, N, K, 22))
    want = rt4.gemm_w8a8(w, sw, x, sx)
    n = ctypes.c_int64()
    L = rt4.lib()
    assert L.rt4_w8a8_work_bytes(M, N, K, 1, ctypes.byref(n)) == 0 and n.value > 0
    work = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    for ptr, size in ((None, 0), (work.data_ptr(), n.value - 1), (work.data_ptr(), n.value)):
        out = torch.zeros(M, N, device="cuda")
        assert L.rt4_gemm_w8a8(out.data_ptr(), N, 0, w.data_ptr(), K, sw.data_ptr(), x.data_ptr(), K, sx.data_ptr(), M, N, K, ptr, size,
                               torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_product_of_extreme_codes(rt4, torch_gpu, M):
    """The longest sums of the largest products come within 2^-13 of the int32 range and are exact."""
    torch = torch_gpu
    K, N = 131056, 70
    x = torch.full((M, K), -128, dtype=torch.int8)
    w = torch.full((N, K), -128, dtype=torch.int8)
    x[0] = 127
    w[1] = 127
    w[2, 1::2] = 127
    one = torch.ones(max(M, N)).cuda()
    got = rt4.gemm_w8a8(w.cuda(), one[:N].contiguous(), x.cuda(), one[:M].contiguous())
    ref = product(torch, x, torch.ones(M), w, torch.ones(N))
    assert float(ref.max()) == 131056 * 16384 or M == 1
    near(torch, got, ref, U, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 70, 256), (3, 200, 144), (50, 130, 400), (300, 270, 336)])
def test_strided_operands(rt4, torch_gpu, M, N, K):
    """Slices of wider matrices: gate and up weights one behind the other, activations among others, output columns of a wider
    row; what lies around the output stays as it is."""
    torch = torch_gpu
    x, sx = codes8(torch, M, K + 64, 6)
    w, sw = codes8(torch, 2 * N, K + 32, 7)
    big = torch.full((M + 2, N + 9), 7.0, device="cuda")
    xs, wd, swd = x.cuda()[:, 16:16 + K], w.cuda(), sw.cuda()
    out = rt4.gemm_w8a8(wd[:N, 16:16 + K], swd[:N], xs, sx.cuda(), out=big[1:M + 1, 4:N + 4])
    ref = product(torch, x[:, 16:16 + K], sx, w[:N, 16:16 + K], sw[:N])
    near(torch, out, ref, 3 * U, torch.float32)
    big[1:M + 1, 4:N + 4] = 7
    assert bool((big == 7).all())
    g, u = ref, product(torch, x[:, 16:16 + K], sx, w[N:, 16:16 + K], sw[N:])
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.full((M + 2, N + 9), 7.0, device="cuda", dtype=dtype)
        out = rt4.ffn_gate_w8a8(wd[:N, 16:16 + K], swd[:N], wd[N:, 16:16 + K], swd[N:], xs, sx.cuda(), out=big[1:M + 1, 5:N + 5])
        near(torch, out, act64(torch, g, "silu") * u, gate_bound(torch, g, "silu"), dtype, gate_flushed(g, u))
        big[1:M + 1, 5:N + 5] = 7
        assert bool((big == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_scales_that_are_not_finite(rt4, torch_gpu, M):
    torch = torch_gpu
    N, K = 200, 256
    x, sx = codes8(torch, M, K, 8)
    w, sw = codes8(torch, N, K, 9)
    x[0, :] = 0
    sw[3], sw[5], sw[7] = math.inf, math.nan, -math.inf
    sx[M - 1] = math.nan if M > 2 else sx[M - 1]
    ref = product(torch, x, sx, w, sw)
    got = rt4.gemm_w8a8(w.cuda(), sw.cuda(), x.cuda(), sx.cuda()).cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fine = torch.isfinite(ref)
    near(torch, got[fine], ref[fine], 3 * U, torch.float32)
    h = rt4.ffn_gate_w8a8(w.cuda(), sw.cuda(), w.cuda(), sw.cuda(), x.cuda(), sx.cuda()).cpu().double()
    want = ref / (1 + torch.exp(-ref)) * ref
    assert torch.equal(torch.isnan(h), torch.isnan(want))


# ------------------------------------------------------------- RT4 gated --
def rt4_case(torch, M, N, K, seed):
    from rt4_amd import layout
    r = np.random.default_rng(seed)
    x = r.standard_normal((M, K)).astype(np.float32)
    if M > 1:
        x[1, :128] = 0
    ws = [(np.abs(r.standard_normal((N, K // 128))) * 0.01 + 1e-3).astype(np.float16) for _ in range(2)]
    wq = [r.integers(0, 2**32, (N, K // 8), dtype=np.uint32) for _ in range(2)]
    codes = [((w[..., None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).astype(np.int64).reshape(N, K) for w in wq]
    codes = [np.where(c > 7, c - 16, c) for c in codes]
    return x, wq, ws, codes, layout


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 37, 256), (2, 100, 640), (3, 17, 1152), (4, 33, 5120), (4, 515, 384), (1, 700, 5120),
                                   (2, 48, 17408), (1, 5, 17408), (3, 1200, 512), (4, 4100, 1024),
                                   (3, 9, 2048), (4, 7, 1152), (2, 3, 896), (1, 2, 3328), (4, 3, 38912)])
def test_gated_half_of_rt4_weights(rt4, torch_gpu, M, N, K, act):
    """Group sums are exact and folded in fp32: each of the K/128 terms carries 3 u and passes through at most K/128 + 8 sums."""
    torch = torch_gpu
    x, wq, ws, codes, layout = rt4_case(torch, M, N, K, N + K)
    dev = lambda a: torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()  # noqa: E731
    xq, sa = rt4.quant_act_a8(dev(x))
    got = rt4.ffn_gate_w4a8(dev(wq[0]), dev(ws[0]), dev(wq[1]), dev(ws[1]), xq, sa, act=act)
    q = layout.deinterleave(xq.cpu().numpy()).astype(np.float64).reshape(M, K // 128, 128) * sa.cpu().numpy().astype(np.float64)[..., None]
    y, size = [], []
    for c, s in zip(codes, ws):
        v = c.astype(np.float64).reshape(N, K // 128, 128) * s.astype(np.float64)[..., None]
        terms = np.einsum("mgk,ngk->mng", q, v)
        y.append(torch.from_numpy(terms.sum(-1)))
        size.append(torch.from_numpy(np.abs(terms).sum(-1)))
    g, u = y
    eps = U * (K // 128 + 11)
    dg, du = eps * size[0], eps * size[1]        # absolute errors of g and u
    want = act64(torch, g, act) * u
    rel = gate_bound(torch, g, act)
    slope = 1.2                                  # |act'| < 1.13 for both
    bound = act64(torch, g, act).abs() * du + slope * dg * u.abs() + slope * dg * du + want.abs() * rel + gate_flushed(g, u) + 2.0 ** -126
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    same = rt4.ffn_gate_w4a8(dev(wq[0]), dev(ws[0].view(np.int16)), dev(wq[1]), dev(ws[1].view(np.int16)), xq, sa, act=act)
    assert torch.equal(got, same)


# ------------------------------------------------------------------ norms --
def rms64(torch, x, eps):
    return torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def right_codes(p, most):
    """Nearest integers (ties to even) to most * p / max|p| over the last axis, with 64 significant bits."""
    p = p.numpy().astype(np.longdouble)
    a = np.abs(p).max(-1, keepdims=True)
    q = np.rint(p * most / np.where(a > 0, a, 1))
    return q.astype(np.int64), a[..., 0].astype(np.float64)


def natural(codes):
    from rt4_amd import layout
    return layout.deinterleave(codes.cpu().numpy()).astype(np.int64)


def expect_form(torch, rt4, out, n, h, w, eps, offset):
    """Checks block_norm's result n of form `out` for residuals h as stored."""
    M, K = h.shape
    h = h.double().cpu()
    p = h * (w.double().cpu() + offset)
    r = rms64(torch, h, eps)
    if not isinstance(n, tuple):
        near(torch, n, p * r, 2 * U if n.dtype is not torch.float32 else 2.0 ** -40, n.dtype)
        return
    q, s = n
    if out == "token":
        codes, a = right_codes(p, 127)
        got, scale = q.cpu().numpy().astype(np.int64), a * r[:, 0].numpy() / 127
    else:
        most = 127 if out == "act" else 119
        codes, a = right_codes(p.reshape(M, K // 128, 128), most)
        got, scale = natural(q), a * r.numpy() / most
        codes = codes.reshape(M, K)
        if out == "rows":
            scale, a = scale.T, a.T
    assert np.array_equal(got, codes), int((got != codes).sum())
    scale = np.where(a > 0, scale, 1.0)
    # (atol: half of fp32's smallest subnormal, what the rounding of a scale below its normal numbers is off by at most)
    np.testing.assert_allclose(s.cpu().numpy(), scale, rtol=2.0 ** -24 * 1.001, atol=2.0 ** -150)


TYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f32", "bf16", "f16", "token", "act", "rows"])
@pytest.mark.parametrize("ht,yt", [("float32", None), ("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float16"),
                                   ("bfloat16", None)])
@pytest.mark.parametrize("M,K", [(1, 128), (3, 5120), (2, 8320), (1100, 256), (1500, 1152), (1, 17408), (2, 65536)])
def test_block_norm(rt4, torch_gpu, M, K, ht, yt, out):
    torch = torch_gpu
    g = torch.Generator().manual_seed(M + K)
    h = (torch.randn((M, K), generator=g) * 3).to(getattr(torch, ht))
    h[:, 5] *= 40
    w = 1 + 0.2 * torch.randn((K,), generator=g)
    y = None if yt is None else torch.randn((M, K), generator=g).to(getattr(torch, yt))
    variants = [(False, None, 0.0)] if y is None else [(False, None, 0.0), (True, "channel", 1.0), (True, None, 0.0), (False, "token", 0.0)]
    for post, gate, offset in variants:
        pw = 1 + 0.2 * torch.randn((K,), generator=g) if post else None
        gt = None if gate is None else torch.rand((K,) if gate == "channel" else (M, K), generator=g).to(y.dtype)
        dev = lambda t: None if t is None else t.cuda()  # noqa: E731
        hn, n = rt4.block_norm(dev(h), dev(y), weight=dev(w), post_weight=dev(pw), gate=dev(gt), scale=0.7, eps=1e-5, weight_offset=offset, out=out)
        if y is not None:
            v = y.double()
            if post:
                v = v * rms64(torch, v, 1e-5) * pw.double()
            if gt is not None:
                v = v * gt.double()
            v = v * 0.7
            want = h.double() + v
            # sums of terms that cancel keep the 64-bit rounding of the larger one, far below a step of the sum unless 2^40 times smaller
            fine = want.abs() > (h.double().abs() + v.abs()) * 2.0 ** -12
            near(torch, hn.cpu()[fine], want[fine], 2 * U if h.dtype is not torch.float32 else 2.0 ** -38, h.dtype)
            assert hn.dtype is h.dtype
        expect_form(torch, rt4, out, n, hn if y is not None else h, w, 1e-5, offset)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 1), (2, 7), (5, 63), (3, 65), (4, 1001), (1100, 131), (1030, 8), (2, 8193), (1, 20001), (2, 65535)])
@pytest.mark.parametrize("out", ["f32", "bf16", "token"])
def test_block_norm_of_odd_rows(rt4, torch_gpu, M, K, out):
    """Row lengths that no vector access divides, strided rows, an update in place, what lies around left as it is."""
    torch = torch_gpu
    g = torch.Generator().manual_seed(7 * M + K)
    wide = torch.randn((M, K + 13), generator=g).cuda()
    y = torch.randn((M, K + 3), generator=g).bfloat16().cuda()
    gate = torch.rand((M, K + 1), generator=g).bfloat16().cuda()
    w = torch.randn((K + 1,), generator=g).cuda()[1:]
    pw = torch.randn((K,), generator=g).cuda()
    before = wide.clone()
    h = wide[:, 5:5 + K]
    hn, n = rt4.block_norm(h, y[:, 1:K + 1], weight=w, post_weight=pw, gate=gate[:, :K], scale=-1.5, h_out=h, out=out)
    assert hn.data_ptr() == h.data_ptr()
    v = y[:, 1:K + 1].double()
    want = before[:, 5:5 + K].double() - 1.5 * (v * rms64(torch, v, 1e-6) * pw.double() * gate[:, :K].double())
    fine = want.abs() > 2.0 ** -12
    near(torch, hn[fine], want[fine], 2.0 ** -36, torch.float32)
    expect_form(torch, rt4, out, n, hn, w, 1e-6, 0.0)
    wide[:, 5:5 + K] = before[:, 5:5 + K]
    assert torch.equal(wide, before)
    r, none = rt4.block_norm(h, y[:, 1:K + 1])
    assert none is None
    near(torch, r, before[:, 5:5 + K].double() + v, U, torch.float32) if bool(((before[:, 5:5 + K].double() + v).abs() > 2.0 ** -10).all()) else None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 16), (4, 17408), (1000, 333), (1200, 2048), (2, 65536), (1, 4097)])
def test_quant_token(rt4, torch_gpu, M, K, dtype):
    torch = torch_gpu
    g = torch.Generator().manual_seed(K)
    x = (torch.randn((M, K), generator=g) * torch.randn((M, K), generator=g)).to(getattr(torch, dtype))
    if M > 1:
        x[1] = 0
    if M > 2:                                    # exact halves: 254 x / max is odd
        x[2, :] = torch.randint(-127, 128, (K,), generator=g).to(x.dtype) / 2
        x[2, 0] = 127
    q, s = rt4.quant_token_a8(x.cuda())
    codes, a = right_codes(x.double(), 127)
    assert np.array_equal(q.cpu().numpy().astype(np.int64), codes)
    np.testing.assert_allclose(s.cpu().numpy(), np.where(a > 0, a / 127, 1.0), rtol=2.0 ** -24 * 1.001, atol=0)
    wide = torch.zeros((M, K + 5), dtype=x.dtype).cuda()
    wide[:, 3:3 + K] = x.cuda()
    q2, s2 = rt4.quant_token_a8(wide[:, 3:3 + K])
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(rt4, torch_gpu, bad):
    """Such a token (or its group) has NaN for a scale and no codes; the others are untouched."""
    torch = torch_gpu
    g = torch.Generator().manual_seed(3)
    h = torch.randn((4, 512), generator=g)
    clean = h.clone()
    h[1, 200] = bad
    w = torch.ones(512)
    q, s = rt4.quant_token_a8(h.cuda())
    q0, s0 = rt4.quant_token_a8(clean.cuda())
    keep = [0, 2, 3]
    assert torch.equal(q[keep], q0[keep]) and torch.equal(s[keep], s0[keep])
    assert bool(s[1].isnan()) and not bool(q[1].any())
    for out in ("token", "act", "rows"):
        _, (q, s) = rt4.block_norm(h.cuda(), weight=w.cuda(), out=out)
        _, (q0, s0) = rt4.block_norm(clean.cuda(), weight=w.cuda(), out=out)
        if out == "rows":
            s, s0 = s.T, s0.T
        assert torch.equal(q[keep], q0[keep]) and torch.equal(s[keep], s0[keep])
        row = s[1].reshape(-1)
        assert bool(row[1 if out != "token" else 0].isnan())
        assert not bool(q[1, 128:256].any())
    _, n = rt4.block_norm(h.cuda(), weight=w.cuda())
    want = h.double() * rms64(torch, h.double(), 1e-6)
    near(torch, n[keep], want[keep], 2.0 ** -38, torch.float32)
    assert torch.equal(n[1].isnan().cpu(), want[1].isnan())
    # a zero token, and weights that are all zeros
    z = torch.zeros((2, 256)).cuda()
    _, (q, s) = rt4.block_norm(z, weight=torch.ones(256).cuda(), out="token")
    assert not bool(q.any()) and bool((s == 1).all())
    _, (q, s) = rt4.block_norm(z + 1, weight=torch.zeros(256).cuda(), out="act")
    assert not bool(q.any()) and bool((s == 1).all())


# ------------------------------------------------------- the block, whole --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("K", [256, 99])
def test_residual_whose_factors_leave_fp32(rt4, torch_gpu, dtype, K):
    """scale * gate * y is formed in fp32 where that decides a 16-bit residual: not where a product on the way underflows, loses
    digits or overflows though the whole does not."""
    torch = torch_gpu
    t = getattr(torch, dtype)
    for scale, yv, gv, hv in ((1e-20, 1e-30, 1e35, 0.0), (1e-20, 1e-30, 1e35, 2e-15), (1e-42, 1e30, 1e12, 0.0), (1e-60, 1e30, 1e30, 1.0), (1e20, 1e30, 1e-37, 5.0),
                              (1e20, 1e30, 0.0, 5.0), (1e40, 0.0, 1.0, 3.0), (1e40, 1e-38, 1.0, 3.0), (1.0, 1e-38, 1.0, 0.0), (0.0, 1e30, 1.0, 2.0)):
        g = torch.Generator().manual_seed(K)
        some = lambda v: (v * (1 + torch.rand((2, K), generator=g)))  # noqa: E731
        h, y, gate = some(hv).to(t), some(yv).float(), some(gv).float()
        got, _ = rt4.block_norm(h.cuda(), y.cuda(), gate=gate.cuda(), scale=scale)
        ref = h.double() + scale * gate.double() * y.double()
        want = ref.float().to(t)
        # ref is off by 2^-51: within that of two neighbours' border, either
        low, high = (ref * (1 - 2.0 ** -50)).float().to(t), (ref * (1 + 2.0 ** -50)).float().to(t)
        ok = (got.cpu() == want) | (got.cpu() == low) | (got.cpu() == high)
        assert bool(ok.all()), (scale, yv, gv, hv, got.cpu()[~ok][:4], want[~ok][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["token", "act", "rows"])
@pytest.mark.parametrize("offset", [0.1, 1.0 / 3.0, 1e-40, 0.5])
def test_codes_whose_weights_nearly_cancel(rt4, torch_gpu, out, offset):
    """weight + offset in 64 bits also where the offset is no fp32 value and the sum is next to nothing."""
    torch = torch_gpu
    M, K = 3, 512
    g = torch.Generator().manual_seed(7)
    h = torch.randn((M, K), generator=g)
    w = (-torch.full((K,), offset, dtype=torch.float64) * (1 + torch.randint(-2, 3, (K,), generator=g) * U)).float()
    got, n = rt4.block_norm(h.cuda(), weight=w.cuda(), weight_offset=offset, out=out)
    expect_form(torch, rt4, out, n, h, w, 1e-6, offset)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [1, 2])
@pytest.mark.parametrize("M", [2, 8, 40, 300])
def test_rows_far_apart(rt4, torch_gpu, M, weights):
    """The largest row strides of codes (offsets within a tile pass 31 bits, rows 32), and outputs whose rows lie as far apart."""
    torch = torch_gpu
    N, K, ld = 300, 272, 2 ** 24 - 16
    x, sx = codes8(torch, M, K, 31)
    w, sw = codes8(torch, N, K, 32)
    far = torch.empty(299 * ld + K, dtype=torch.int8, device="cuda")
    xf, wf = far.as_strided((M, K), (ld, 1), 0), far.as_strided((N, K), (ld, 1), 0)
    o = torch.empty(299 * 2 ** 23 + N, dtype=torch.bfloat16, device="cuda").as_strided((M, N), (2 ** 23, 1), 0)
    xf.copy_(x)
    args = (w.cuda(), sw.cuda(), sx.cuda())
    if weights == 1:
        want = rt4.gemm_w8a8(args[0], args[1], x.cuda(), args[2], dtype=torch.bfloat16)
        assert torch.equal(rt4.gemm_w8a8(args[0], args[1], xf, args[2], out=o), want)
        wf.copy_(w)
        assert torch.equal(rt4.gemm_w8a8(wf, args[1], x.cuda(), args[2], out=o), want)
    else:
        want = rt4.ffn_gate_w8a8(args[0], args[1], args[0], args[1], x.cuda(), args[2], dtype=torch.bfloat16)
        assert torch.equal(rt4.ffn_gate_w8a8(args[0], args[1], args[0], args[1], xf, args[2], out=o), want)
        wf.copy_(w)
        assert torch.equal(rt4.ffn_gate_w8a8(args[0], args[1], wf, args[1], x.cuda(), args[2], out=o), want)


@pytest.mark.gpu
def test_wide_decode_half_captured(rt4, torch_gpu):
    """Four rows whose codes need more LDS than a launch is granted without asking, captured and replayed."""
    torch = torch_gpu
    rows, N, K = 4, 70, 20480
    g = torch.Generator().manual_seed(3)
    w = [torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), generator=g, dtype=torch.int64).to(torch.int32).cuda() for _ in range(2)]
    s = [(torch.rand((N, K // 128), generator=g) * 0.01).to(torch.float16).cuda() for _ in range(2)]
    x = torch.randn((rows, K), generator=g).cuda()

    def run():
        return rt4.ffn_gate_w4a8(w[0], s[0], w[1], s[1], *rt4.block_norm(x, weight=torch.ones(K, device="cuda"), out="act")[1])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(3):
        x.copy_(torch.randn((rows, K), generator=g))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def ffn_block(rt4, h, y, p):
    """One feed-forward block at 8 bits: norm and quantize, gated half, quantize, down, and the residual normed for the next block."""
    h1, (xq, sx) = rt4.block_norm(h, y, weight=p["w1"], post_weight=p["pw"], scale=0.5, out="token")
    a = rt4.ffn_gate_w8a8(p["wg"], p["sg"], p["wu"], p["su"], xq, sx, dtype=h.dtype)
    aq, sa = rt4.quant_token_a8(a)
    d = rt4.gemm_w8a8(p["wd"], p["sd"], aq, sa, dtype=h.dtype)
    h2, n = rt4.block_norm(h1, d, weight=p["w2"], out="bf16")
    return h1, xq, sx, a, aq, sa, d, h2, n


def ffn_case(torch, M, D, F, dtype):
    g = torch.Generator().manual_seed(M)
    p = {"w1": 1 + 0.1 * torch.randn(D, generator=g), "w2": 1 + 0.1 * torch.randn(D, generator=g), "pw": 1 + 0.1 * torch.randn(D, generator=g)}
    for k, (n, kk) in {"g": (F, D), "u": (F, D), "d": (D, F)}.items():
        q, s = codes8(torch, n, kk, ord(k))
        p["w" + k], p["s" + k] = q, s / math.sqrt(kk)
    return torch.randn((M, D), generator=g).to(dtype), torch.randn((M, D), generator=g).to(dtype), p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M", [1, 4, 37, 300])
def test_feed_forward_block(rt4, torch_gpu, M, dtype):
    """Each step against its definition on what the step before it gave."""
    torch = torch_gpu
    dtype = getattr(torch, dtype)
    h, y, p = ffn_case(torch, M, 640, 1104, dtype)
    c = {k: v.cuda() for k, v in p.items()}
    h1, xq, sx, a, aq, sa, d, h2, n = ffn_block(rt4, h.cuda(), y.cuda(), c)
    e = 1e-6
    expect_form(torch, rt4, "token", (xq, sx), h1, p["w1"], e, 0.0)
    g, u = (product(torch, xq.cpu(), sx.cpu(), p["w" + k], p["s" + k]) for k in "gu")
    near(torch, a, act64(torch, g, "silu") * u, gate_bound(torch, g, "silu"), dtype, gate_flushed(g, u))
    codes, m = right_codes(a.double().cpu(), 127)
    assert np.array_equal(aq.cpu().numpy().astype(np.int64), codes)
    near(torch, d, product(torch, aq.cpu(), sa.cpu(), p["wd"], p["sd"]), 3 * U, dtype)
    expect_form(torch, rt4, "bf16", n, h2, p["w2"], e, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_block_captured_and_replayed(rt4, torch_gpu, M):
    """A captured block on new inputs gives, at every replay, what the eager one gives, bit for bit."""
    torch = torch_gpu
    h, y, p = ffn_case(torch, M, 640, 1104, torch.bfloat16)
    c = {k: v.cuda() for k, v in p.items()}
    h, y = h.cuda(), y.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ffn_block(rt4, h, y, c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ffn_block(rt4, h, y, c)
    for i in range(4):
        h.copy_(torch.randn_like(h))
        y.copy_(torch.randn_like(y))
        want = ffn_block(rt4, h, y, c)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_blocks_on_two_streams(rt4, torch_gpu, M):
    """Calls on two streams share nothing: both give what they give alone."""
    torch = torch_gpu
    cases = []
    for i in range(2):
        h, y, p = ffn_case(torch, M + i, 640, 1104, torch.bfloat16)
        cases.append((h.cuda(), y.cuda(), {k: v.cuda() for k, v in p.items()}))
    want = [ffn_block(rt4, *c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [None, None]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = ffn_block(rt4, *cases[i])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for s, t in zip(a, b):
                assert torch.equal(s, t)


@pytest.mark.gpu
def test_decode_block_of_rt4_weights(rt4, torch_gpu):
    """block_norm's group codes feed the RT4 linears: the same layout that quant_act_a8 and quant_rows_i8 write, and a result that
    differs from theirs by codes next to a border alone."""
    torch = torch_gpu
    M, K = 4, 1280
    g = torch.Generator().manual_seed(11)
    h, w = torch.randn((M, K), generator=g).cuda(), (1 + 0.1 * torch.randn(K, generator=g)).cuda()
    _, n = rt4.block_norm(h, weight=w)
    _, (q, s) = rt4.block_norm(h, weight=w, out="act")
    q0, s0 = rt4.quant_act_a8(n)
    assert q.shape == q0.shape and s.shape == s0.shape
    assert int((q.int() - q0.int()).abs().max()) <= 1 and int((q != q0).sum()) <= 5
    assert float(((s - s0) / s0).abs().max()) < 4 * U
    _, (q, s) = rt4.block_norm(h, weight=w, out="rows")
    q0, s0 = rt4.quant_rows_i8(n)
    assert q.shape == q0.shape and s.shape == s0.shape
    assert int((q.int() - q0.int()).abs().max()) <= 1 and int((q != q0).sum()) <= 5
    assert float(((s - s0) / s0).abs().max()) < 4 * U


# --------------------------------------------------------------- refusals --
def test_product_refusals(rt4):
    L = rt4.lib()

    def call(c=DUMMY, ldc=64, t=0, w=DUMMY, ldw=256, sw=DUMMY, x=DUMMY, ldx=256, sx=DUMMY, M=4, N=64, K=256):
        return L.rt4_gemm_w8a8(c, ldc, t, w, ldw, sw, x, ldx, sx, M, N, K, None, 0, None)

    for name in ("c", "w", "sw", "x", "sx"):
        assert call(**{name: None}) == 2
    for kw in ({"M": 0}, {"N": 0}, {"M": -1}, {"K": 0}, {"K": 8}, {"K": 250}, {"K": 131072, "ldx": 131072, "ldw": 131072}, {"ldc": 63}, {"ldx": 240},
               {"ldx": 264}, {"ldw": 255}, {"ldw": 1 << 24}, {"M": (1 << 24) + 1}, {"N": (1 << 24) + 1},
               {"M": 1 << 24, "N": 1 << 24, "ldc": 1 << 24}):
        assert call(**kw) == 1, kw
        assert "rt4_gemm_w8a8" in L.rt4_last_error().decode()
    for kw in ({"t": 3}, {"t": -1}, {"w": ODD}, {"x": ODD}, {"c": ctypes.c_void_p(0x1002)}, {"sx": ctypes.c_void_p(0x1002)}):
        assert call(**kw) == 2, kw


def test_sizes_beyond_a_launch(rt4):
    """What a grid of workgroups cannot count is refused."""
    L = rt4.lib()
    assert L.rt4_gemm_w8a8(DUMMY, 2 ** 14, 1, DUMMY, 16, DUMMY, DUMMY, 16, DUMMY, 2 ** 24, 2 ** 14, 16, None, 0, None) == 1
    assert L.rt4_w8a8_work_bytes(2 ** 24, 2 ** 14, 16, 1, ctypes.byref(ctypes.c_int64())) == 1
    for M, N in ((2 ** 24, 2 ** 13), (2 ** 13, 2 ** 24), (2 ** 24, 33), (9, 2 ** 24)):
        for weights in (1, 2):
            for p in rt4.w8a8_launch_plan(M, N, 16, weights, cus=256):
                tiles = -(-M // p["tile_m"]) * -(-p["channels"] // (p["tile_n"] // weights))
                assert tiles * p["splits"] * 256 < 2 ** 32
    assert L.rt4_quant_token_a8(DUMMY, DUMMY, DUMMY, 1, 1, 2 ** 22, 1, None) == 1
    assert L.rt4_block_norm(None, 0, DUMMY, 16, 1, None, 0, 0, None, 0, None, DUMMY, 1.0, 1e-6, 0.0, DUMMY, None, 1, 2 ** 22, 16, None) == 1


def test_plan_refusals(rt4):
    for args in ((0, 64, 256, 1), (4, 0, 256, 1), (4, 64, 24, 1), (4, 64, 131072, 1), (4, 64, 256, 0), (4, 64, 256, 3)):
        with pytest.raises(rt4.RT4Error):
            rt4.w8a8_launch_plan(*args, cus=256)
    with pytest.raises(rt4.RT4Error):
        rt4.w8a8_launch_plan(4, 64, 256, 1, cus=-1)
    assert rt4.lib().rt4_w8a8_work_bytes(4, 64, 24, 1, ctypes.byref(ctypes.c_int64())) == 1
    assert rt4.lib().rt4_w8a8_work_bytes(4, 64, 256, 1, None) == 2


def test_gated_refusals(rt4):
    L = rt4.lib()

    def call(h=DUMMY, ldh=64, t=1, wg=DUMMY, ldg=256, sg=DUMMY, wu=DUMMY, ldu=256, su=DUMMY, x=DUMMY, ldx=256, sx=DUMMY, M=4, N=64, K=256, act=0):
        return L.rt4_ffn_gate_w8a8(h, ldh, t, wg, ldg, sg, wu, ldu, su, x, ldx, sx, M, N, K, act, None, 0, None)

    for name in ("h", "wg", "sg", "wu", "su", "x", "sx"):
        assert call(**{name: None}) == 2
    for kw in ({"M": 0}, {"N": 0}, {"K": 24}, {"ldh": 1}, {"ldu": 128}, {"ldg": 260}):
        assert call(**kw) == 1, kw
    for kw in ({"act": 2}, {"act": -1}, {"t": 5}, {"wu": ODD}):
        assert call(**kw) == 2, kw

    def call4(h=DUMMY, wg=DUMMY, sg=DUMMY, wu=DUMMY, su=DUMMY, x=DUMMY, sa=DUMMY, rows=4, N=64, K=256, act=0):
        return L.rt4_ffn_gate_w4a8(h, wg, sg, wu, su, x, sa, rows, N, K, act, None)

    for name in ("h", "wg", "sg", "wu", "su", "x", "sa"):
        assert call4(**{name: None}) == 2
    for kw in ({"rows": 0}, {"rows": 5}, {"K": 200}, {"K": 0}, {"N": 0}):
        assert call4(**kw) == 1, kw
    for kw in ({"act": 2}, {"wu": ODD}, {"x": ODD}):
        assert call4(**kw) == 2, kw


def test_norm_refusals(rt4):
    L = rt4.lib()

    def call(ho=DUMMY, ldho=256, h=ctypes.c_void_p(0x2000), ldh=256, ht=0, y=DUMMY, ldy=256, yt=0, gate=None, ldg=0, pw=None, w=DUMMY, scale=1.0, eps=1e-6,
             off=0.0, n=DUMMY, ns=DUMMY, form=3, M=4, K=256):
        return L.rt4_block_norm(ho, ldho, h, ldh, ht, y, ldy, yt, gate, ldg, pw, w, scale, eps, off, n, ns, form, M, K, None)

    for kw in ({"h": None}, {"ho": None}, {"w": None}, {"n": None}, {"ns": None}, {"form": 6}, {"form": -1}, {"ht": 3}, {"yt": -1}, {"eps": -1.0},
               {"eps": math.nan}, {"y": None, "n": None, "w": None}, {"y": None, "gate": DUMMY}, {"y": None, "pw": DUMMY}, {"ho": ODD, "h": ODD, "ldh": 300},
               {"n": ODD, "form": 4}, {"h": ctypes.c_void_p(0x2002)}, {"y": ctypes.c_void_p(0x1001), "yt": 1}):
        assert call(**kw) == 2, kw
    for kw in ({"M": 0}, {"K": 0}, {"K": 65537, "ldh": 70000, "ldy": 70000, "ldho": 70000}, {"ldh": 255}, {"ldy": 255}, {"ldho": 0},
               {"gate": DUMMY, "ldg": 100}, {"form": 4, "K": 200}, {"form": 5, "K": 136}):
        assert call(**kw) == 1, kw

    def quant(q=DUMMY, s=DUMMY, x=DUMMY, ldx=256, t=0, M=4, K=256):
        return L.rt4_quant_token_a8(q, s, x, ldx, t, M, K, None)

    for kw in ({"q": None}, {"s": None}, {"x": None}, {"t": 7}, {"x": ctypes.c_void_p(0x1001), "t": 1}):
        assert quant(**kw) == 2, kw
    for kw in ({"M": 0}, {"K": 0}, {"ldx": 255}, {"K": 65537, "ldx": 65537}):
        assert quant(**kw) == 1, kw


@pytest.mark.gpu
def test_wrapper_refusals(rt4, torch_gpu):
    torch = torch_gpu
    x, sx = codes8(torch, 4, 256, 1)
    w, sw = codes8(torch, 8, 256, 2)
    x, sx, w, sw = x.cuda(), sx.cuda(), w.cuda(), sw.cuda()
    h = torch.randn(4, 256).cuda()
    one = torch.ones(256).cuda()
    for fn in (lambda: rt4.gemm_w8a8(w.cpu(), sw, x, sx), lambda: rt4.gemm_w8a8(w, sw[:7], x, sx), lambda: rt4.gemm_w8a8(w, sw, x.int(), sx),
               lambda: rt4.gemm_w8a8(w, sw, x, sx.double()), lambda: rt4.gemm_w8a8(w, sw, x, sx, dtype=torch.int32), lambda: rt4.gemm_w8a8(w[:, :128], sw, x, sx),
               lambda: rt4.gemm_w8a8(w, sw, x.T, sx), lambda: rt4.gemm_w8a8(w, sw, x, sx, out=torch.empty(4, 9).cuda()),
               lambda: rt4.gemm_w8a8(w, sw, x, sx, out=torch.empty(4, 8).cuda(), dtype=torch.bfloat16), lambda: rt4.gemm_w8a8(w[:, 1:129], sw, x[:, 1:129], sx),
               lambda: rt4.ffn_gate_w8a8(w, sw, w[:7], sw, x, sx), lambda: rt4.ffn_gate_w8a8(w, sw, w, sw, x, sx, act="relu"),
               lambda: rt4.gemm_w8a8(w, sw, x[:0], sx[:0]), lambda: rt4.block_norm(h), lambda: rt4.block_norm(h, weight=one, out="int8"),
               lambda: rt4.block_norm(h, weight=one[:255]), lambda: rt4.block_norm(h, gate=one, weight=one), lambda: rt4.block_norm(h, h.half(), gate=one, weight=one),
               lambda: rt4.block_norm(h, h_out=h, weight=one), lambda: rt4.block_norm(h[:, ::2], weight=one[:128]), lambda: rt4.block_norm(h.double(), weight=one),
               lambda: rt4.block_norm(h, h[:3], weight=one), lambda: rt4.quant_token_a8(h.long()), lambda: rt4.quant_token_a8(h[0]),
               lambda: rt4.quant_token_a8(h, xq=torch.empty(4, 255, dtype=torch.int8).cuda())):
        with pytest.raises(rt4.RT4Error):
            fn()


@pytest.mark.gpu
def test_rows_beyond_32_bits_are_refused(rt4, torch_gpu):
    """More rows than the C ABI's ints hold: refused, not cut."""
    torch = torch_gpu
    x = torch.empty((2 ** 32 + 1, 1), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(rt4.RT4Error):
        rt4.quant_token_a8(x)
    with pytest.raises(rt4.RT4Error):
        rt4.block_norm(x, weight=torch.ones(1, device="cuda"))
