"""Device arrays of any contents in calls large enough for sums of them to pass 32 bits: nothing outside the call's
memory is touched, and the call comes back."""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import paged8
from test_paged8_gpu import make_pools

pytestmark = pytest.mark.gpu
D = 64
GUARD = 1 << 20


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_overlapping_rows_that_cost_more_than_the_line_holds(dev, code, monkeypatch):
    """64 rows, every other of all 8192 tokens behind 130000 slots: 2.2e9 by the count that even pieces are cut by."""
    gen = torch.Generator().manual_seed(21)
    b, kvh, g, total, page = 64, 2, 16, 8192, 4096
    layer = tuple(t[0] for t in make_pools(gen, 3, kvh, page, code, dev))
    before = [t.clone() for t in layer]
    # Slots up to 118784 in two pages, taken in turn; none for the new tokens.
    table = (torch.arange(32, dtype=torch.int32) % 2).repeat(b, 1)
    table[:, 29:] = -1
    table = table.to(dev)
    x = torch.randn(total, (g + 2) * kvh, D, generator=gen).half().to(dev)
    cu = torch.tensor([0 if r % 2 == 0 else total for r in range(b + 1)], dtype=torch.int32, device=dev)
    ctx = torch.full((b,), 130000, device=dev)
    taken = []

    def scratch(need, device):
        taken.append(torch.full((need + 2 * GUARD,), 0x5A, device=device, dtype=torch.uint8))
        return taken[-1][GUARD:GUARD + need]

    monkeypatch.setattr(paged8, "_scratch", scratch)
    out = paged8.prefill_extend_paged8(x[:, :g * kvh], x[:, g * kvh:(g + 1) * kvh], x[:, (g + 1) * kvh:], cu, total, ctx,
                                       None, None, layer, table, lengths=[total // b] * b)
    torch.cuda.synchronize()
    assert out.shape == (total, g * kvh, D) and len(taken) == 1
    assert bool((taken[0][:GUARD] == 0x5A).all()) and bool((taken[0][-GUARD:] == 0x5A).all())
    for t, u in zip(layer, before):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))
    monkeypatch.undo()
    # The next call over the same pages is right.
    q = torch.randn(1, kvh, g, D, generator=gen).half().to(dev)
    got = paged8.flash_decode_attention_paged8(q, layer, table[:1], torch.tensor([299], device=dev))
    cu = torch.tensor([0, 300], dtype=torch.int32, device=dev)
    k, v = (t.double().cpu().numpy() for t in paged8.read_paged8(layer, table[:1], cu, 300,
                                                                 torch.zeros(1, dtype=torch.int64, device=dev)))
    want = kv8.attend(q.reshape(-1, D).cpu().double().numpy(), k, v)
    # Weights off by 2^-11 each way and the output by 2^-11 of the largest value, fp32 sums beside them.
    assert np.abs(got.reshape(-1, D).cpu().double().numpy() - want).max() <= 3.1 * 2.0 ** -11 * np.abs(v).max()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_rows_of_two_to_the_31_slots(dev, code):
    """The longest rows that the calls take, all of one page: their slots' mean is the page's."""
    page, ppr = 4096, 524287
    kv = paged8.PagedKv8Cache(1, 1, 1, page, 1, 1, dev, code)
    one = torch.ones(page, 1, D, device=dev, dtype=torch.float16)
    cu = torch.tensor([0, page], dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    table = torch.zeros(1, ppr, dtype=torch.int32, device=dev)
    paged8.append_paged8(0 * one, one, cu, page, zero, None, None, kv.pools[0], table[:, :1].contiguous())
    q = torch.randn(2, 3, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    last = torch.tensor([page * ppr - 1], device=dev)
    got = paged8.flash_decode_attention_paged8(q[:1, None], kv.pools[0], table, last)
    assert torch.equal(got, torch.ones_like(got))
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    got = paged8.prefill_extend_paged8(q, 0 * one[:2], one[:2], cu, 2, last - 1, None, None, kv.pools[0], table)
    assert torch.equal(got, torch.ones_like(got))
