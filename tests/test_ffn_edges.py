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
