"""Factors of the scores down to the least there are, over caches held in 8 bits: all weights alike, masked slots none."""

import pytest
import torch

from qwenforge_amd import paged8

pytestmark = pytest.mark.gpu
D = 64


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [1e-20, 1e-37, 1e-42, 1e-300])
@pytest.mark.parametrize("zero", [True, False])
def test_tiny_factors(dev, code, scale, zero):
    """Values of whole numbers up to 3 over 2^n slots: their mean, bit for bit but for its rounding."""
    gen = torch.Generator().manual_seed(9)
    n = 128
    kv = paged8.PagedKv8Cache(1, 2, 4, 64, 1, 4, dev, code)
    kv.map_row(0, 200)
    k = torch.zeros(n, 2, D) if zero else torch.randn(n, 2, D, generator=gen)
    v = torch.randint(-3, 4, (n, 2, D), generator=gen)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    first = torch.zeros(1, dtype=torch.int64, device=dev)
    paged8.append_paged8(k.half().to(dev), v.half().to(dev), cu, n, first, None, None, kv.pools[0], kv.table)
    q = torch.randn(1, 2, 7, D, generator=gen).half().to(dev)
    for m in (1, 17, 64, 100, 128):
        got = paged8.flash_decode_attention_paged8(q, kv.pools[0], kv.table, first + m - 1, scale=scale)
        want = v[:m].double().mean(dim=0)[:, None].expand(-1, 7, -1)
        assert ((got[0].double().cpu() - want).abs() <= (2.0 ** -11 + 2.0 ** -22) * want.abs()).all(), m
    new = (q.view(1, 14, D), k[:1].half().to(dev), v[:1].half().to(dev))
    got = paged8.prefill_extend_paged8(*new, cu[:2] // n, 1, first + n, None, None, kv.pools[0], kv.table, scale=scale)
    want = torch.cat([v, v[:1]]).double().mean(dim=0)[:, None].expand(-1, 7, -1)
    assert ((got.view(2, 7, D).double().cpu() - want).abs() <= (2.0 ** -11 + 2.0 ** -22) * want.abs()).all()
