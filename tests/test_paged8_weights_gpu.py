"""Small weights beside a large one, over caches held in 8 bits: one slot far above thousands of others whose weights
matter together.

Tolerance: weights are rounded to fp16 as multiples of at most 2^-7 of the largest that a state has seen, so that one
is off by 2^-11 of itself or, where that is less than 2^-21 of the largest, by 2^-32 of it: the output by 2^-32 of the
sum of all values.  3.1 * 2^-11 relative is the weights' rounding, twice, and the output's, with room for fp32 sums."""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import paged8
from test_paged8_attn_gpu import values_of
from test_paged8_gpu import make_pools, make_table

pytestmark = pytest.mark.gpu
D = 64


def sink_rows(n, kvh):
    """Slot 0 scores 17.7 with a query of 16 in dimension 0, the others 0: e^-17.7 is just below 2^-25."""
    k, v = torch.zeros(n, kvh, D), torch.full((n, kvh, D), 1000.0)
    k[0, :, 0] = 8.85
    v[0] = 0.0
    return k.half(), v.half()


def check(got, q, k, v, what):
    want = kv8.attend(q, k, v)
    bound = 3.1 * 2.0 ** -11 * np.abs(want) + 2.0 ** -32 * np.repeat(np.abs(v).sum(axis=0), len(q) // v.shape[1], axis=0)
    off = np.abs(got.cpu().double().numpy() - want)
    assert (off <= bound).all(), (what, off.max(), bound.min(), want.max())


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("n,ppr", [(1000, 16), (1000, 40), (30000, 470)])
def test_decode(dev, code, n, ppr):
    gen = torch.Generator().manual_seed(3)
    layer = tuple(t[0] for t in make_pools(gen, ppr, 2, 64, code, dev))
    table, host = make_table(gen, [n], 64, ppr, ppr, dev)
    k, v = sink_rows(n, 2)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    paged8.append_paged8(k.to(dev), v.to(dev), cu, n, torch.zeros(1, dtype=torch.int64, device=dev), None, None, layer,
                         table, lengths=[n])
    q = torch.zeros(1, 2, 7, D, dtype=torch.float16, device=dev)
    q[..., 0] = 16.0
    got = paged8.flash_decode_attention_paged8(q, layer, table, torch.tensor([n - 1], device=dev))
    check(got.reshape(-1, D), q.reshape(-1, D).cpu().double().numpy(), *values_of(layer, host[0], n), n)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh,g", [
    ([400], [5000], 8, 16),           # 128 query rows a unit, over all slots
    ([600], [9000], 8, 7),            # the same, in even pieces
    ([300], [2000], 2, 7),            # 32 query rows, in eight waves
    ([300, 300], [3000, 3000], 8, 7), # 48
    ([3], [1500], 2, 7),
])
def test_extension(dev, code, lens, ctx, kvh, g):
    gen = torch.Generator().manual_seed(5)
    need = [c + n for c, n in zip(ctx, lens)]
    n_pages = sum(-(-n // 64) for n in need)
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, 64, code, dev))
    table, host = make_table(gen, need, 64, n_pages, -(-max(need) // 64), dev)
    k, v = sink_rows(max(need), kvh)

    def packed(t, spans):
        return torch.cat([t[a:b] for a, b in spans]).to(dev)

    def starts(n):
        return torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=dev)

    old, new = [(0, c) for c in ctx], list(zip(ctx, need))
    paged8.append_paged8(packed(k, old), packed(v, old), starts(ctx), max(ctx),
                         torch.zeros(len(ctx), dtype=torch.int64, device=dev), None, None, layer, table, lengths=ctx)
    q = torch.zeros(sum(lens), kvh * g, D, dtype=torch.float16, device=dev)
    q[..., 0] = 16.0
    got = paged8.prefill_extend_paged8(q, packed(k, new), packed(v, new), starts(lens), max(lens),
                                       torch.tensor(ctx, device=dev), None, None, layer, table, lengths=lens)
    for r, (n, c) in enumerate(zip(lens, ctx)):
        kk, vv = values_of(layer, host[r], c + n)
        for i in (0, n - 1):
            t = sum(lens[:r]) + i
            check(got[t], q[t].cpu().double().numpy(), kk[:c + i + 1], vv[:c + i + 1], (r, i))
