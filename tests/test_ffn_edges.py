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
