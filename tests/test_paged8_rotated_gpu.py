"""Extensions over caches held in 8 bits that rotate queries and keys themselves: bit for bit the call with queries and
keys rotated before it, in the pages and in the outputs, in every form of the attention."""

import pytest
import torch

from qwenforge_amd import ops, paged8
from test_paged8_attn_gpu import fill_rows
from test_paged8_gpu import make_pools, make_table

pytestmark = pytest.mark.gpu
D = 64


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh,g,slots", [
    ([1, 2, 2, 0, 1], [14, 15, 30, 3, 900], 2, 7, 1024),            # appended by the attention, 16 query rows
    ([4, 1, 3], [1000, -1, 17], 3, 8, 1024),                        # 32
    ([3] * 40, [i * 17 % 900 for i in range(40)], 2, 16, 1024),     # 48
    ([5, 4], [300, 2011], 2, 7, 2048),                              # by a launch of its own, 16 query rows a unit
    ([40, 9], [2500, 2100], 2, 7, 2560),                            # 32, in pieces
    ([300, 250], [3000, 2500], 8, 7, 3328),                         # 48
    ([200, 0, 213], [0, 3, 1000], 16, 8, 1280),                     # 128
    ([300, 40, 250], [6000, -1, 9000], 8, 7, 9280),                 # 128, in even pieces
])
def test_rotated_by_the_call_and_before_it(dev, lens, ctx, kvh, g, slots, code):
    gen = torch.Generator().manual_seed(40 + len(lens) + g)
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // 64) for n in need) + 2
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, 64, code, dev))
    table, _ = make_table(gen, need, 64, n_pages, slots // 64, dev)
    fill_rows(gen, layer, table, ctx, dev)
    other = tuple(t.clone() for t in layer)
    n = sum(lens)
    qkv = torch.randn(n, (g + 2) * kvh, D, generator=gen).half().to(dev)
    q, k, v = qkv[:, :g * kvh], qkv[:, g * kvh:(g + 1) * kvh], qkv[:, (g + 1) * kvh:]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    at = torch.tensor(ctx, device=dev)
    ang = torch.rand(n, 32, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], dim=1).half().to(dev) for f in (torch.cos, torch.sin))
    cache = torch.zeros(n, kvh, 64, D, device=dev, dtype=torch.float16)
    turned = ops.rope_append(q[:, :, None].contiguous(), k[:, :, None].contiguous(), v[:, :, None].contiguous(),
                             cos.view(n, 1, D), sin.view(n, 1, D), cache, cache.clone(),
                             torch.zeros(1, dtype=torch.int64, device=dev))
    got = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), at, cos, sin, layer, table, lengths=lens)
    want = paged8.prefill_extend_paged8(turned[:, :, 0], cache[:, :, 0], v, cu, max(lens), at, None, None, other, table,
                                        lengths=lens)
    assert torch.equal(got, want) and bool(got.any())
    for a, b in zip(layer, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
