"""Rows that are longer on the device than the call's ``max_seqlen`` (their offsets written after the host's check, as
under a replayed graph): every form takes their first ``max_seqlen`` tokens and no others."""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import paged8
from test_paged8_attn_gpu import fill_rows, values_of
from test_paged8_gpu import make_pools, make_table

pytestmark = pytest.mark.gpu
D = 64


def rows_of(gen, code, dev, kvh, ctx, n, page, ppr):
    layer = tuple(t[0] for t in make_pools(gen, 8, kvh, page, code, dev))
    table, host = make_table(gen, [ctx + n, 64], page, 8, ppr, dev)
    fill_rows(gen, layer, table, [ctx, 0], dev)
    # Tokens past max_seqlen are far larger: written, they would change their blocks' scales.
    x = torch.randn(n, 2 * kvh, D, generator=gen)
    x[3:] *= 100
    return layer, table, host, x.half().to(dev)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("longest", [1, 3])
@pytest.mark.parametrize("ctx", [0, 14])
def test_append(dev, code, longest, ctx):
    gen = torch.Generator().manual_seed(3 + ctx)
    layer, table, host, x = rows_of(gen, code, dev, 2, ctx, 40, 64, 2)
    want = tuple(t.clone() for t in layer)
    at = torch.tensor([ctx, 0], device=dev)
    lengths = [1] * 40 if longest == 1 else [3] * 13 + [1]
    b = len(lengths)
    cu = torch.tensor([0, 40] + [40] * (b - 1), dtype=torch.int32, device=dev)    # on the device: one row of them all
    wide = torch.full((b, 2), -1, dtype=torch.int32, device=dev)
    wide[:2] = table
    paged8.append_paged8(x[:, :2], x[:, 2:], cu, longest, torch.cat([at, at.new_zeros(b - 2)]), None, None, layer, wide,
                         lengths=lengths)
    paged8.append_paged8(x[:longest, :2], x[:longest, 2:], torch.tensor([0, longest, longest], dtype=torch.int32, device=dev),
                         longest, at, None, None, want, table)
    for t, u in zip(layer, want):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kvh,g,ppr", [
    (2, 7, 2),        # appended by the attention
    (2, 7, 40),       # by a launch before it
    (2, 16, 2),
])
@pytest.mark.parametrize("ctx", [0, 14])
def test_extension(dev, code, kvh, g, ppr, ctx):
    gen = torch.Generator().manual_seed(5 + ctx + g)
    layer, table, host, x = rows_of(gen, code, dev, kvh, ctx, 5, 64, ppr)
    want = tuple(t.clone() for t in layer)
    q = torch.randn(5, kvh * g, D, generator=gen).half().to(dev)
    at = torch.tensor([ctx, 0], device=dev)
    got = paged8.prefill_extend_paged8(q, x[:, :kvh], x[:, kvh:], torch.tensor([0, 5, 5], dtype=torch.int32, device=dev), 3,
                                       at, None, None, layer, table, lengths=[3, 2])
    paged8.append_paged8(x[:3, :kvh], x[:3, kvh:], torch.tensor([0, 3, 3], dtype=torch.int32, device=dev), 3, at, None,
                         None, want, table)
    for t, u in zip(layer, want):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))
    k, v = values_of(layer, host[0], ctx + 3)
    for i in range(3):
        out = kv8.attend(q[i].cpu().double().numpy(), k[:ctx + i + 1], v[:ctx + i + 1])
        # A weight is off by 2^-11 each way, the output by 2^-11 of the largest value; fp32 sums beside them.
        assert np.abs(got[i].cpu().double().numpy() - out).max() <= 3.1 * 2.0 ** -11 * np.abs(v).max()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("longest", [1, 3])
def test_read(dev, code, longest, monkeypatch):
    """What lies past a row's max_seqlen is left as it was, as tokens of no row are."""
    gen = torch.Generator().manual_seed(7)
    layer, table, host, x = rows_of(gen, code, dev, 2, 40, 5, 64, 2)
    lengths = [1] * 10 if longest == 1 else [3, 3, 3, 1]
    b = len(lengths)
    wide = torch.full((b, 2), -1, dtype=torch.int32, device=dev)
    wide[:2] = table
    first = torch.full((b,), 14, device=dev)
    cu = torch.tensor([0, 10] + [10] * (b - 1), dtype=torch.int32, device=dev)
    plain = torch.empty
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", lambda *a, **kw: plain(*a, **kw).fill_(7.0))
        k, v = paged8.read_paged8(layer, wide, cu, longest, first, lengths=lengths)
    have = paged8.read_paged8(layer, table[:1], torch.tensor([0, longest], dtype=torch.int32, device=dev), longest, first[:1])
    for t, u in zip((k, v), have):
        assert torch.equal(t[:longest], u) and bool((t[longest:] == 7.0).all())
