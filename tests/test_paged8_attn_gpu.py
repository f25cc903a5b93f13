"""Attention over caches held in 8 bits against the definition in 64 bits, over the
values that the pages hold.

Tolerance: the output is sum_j w_j v_j with |v| <= V, v exact in fp16.  The kernel rounds
each p_j to fp16 (half a step, 2^-11) and divides by the sum of the rounded ones, so a
weight is off by at most 2 * 2^-11 relative and the output by 2 * 2^-11 V; p below
fp16's normal range (2^-14 of a reference that is at most 2^8 below the row's largest) is
off by half a step of 2^-24, together at most n * 2^-25 V over a sum of at least 2^-8 --
2^-17 n V, less than 0.02 * 2^-11 V per 64 slots only where that many lie so low, which
random scores within +-16 do not do.  The fp16 output adds 2^-11 V.  Scores are fp32 sums
of 64 products: 64 * 2^-24 * sum |q k| / 8 < 2^-15 for the sizes here, which moves p by as
much.  In all 3.1 * 2^-11 V with room for the fp32 sums of p and p v.
"""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import ops, paged8
from test_paged8_gpu import make_pools, make_table, row_state, spread

pytestmark = pytest.mark.gpu
TOL = 3.1 * 2.0 ** -11
D = 64


def fill_rows(gen, layer, table, rows, dev, size=1.0):
    """K and V of the rows' slots appended (random), everything else left as it was."""
    lens = [max(n, 0) for n in rows]
    kvh = layer[0].shape[1]
    if sum(lens) == 0:
        return
    x = (torch.randn(sum(lens), 2 * kvh, D, generator=gen) * size).half().to(dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    paged8.append_paged8(x[:, :kvh], x[:, kvh:], cu, max(lens),
                         torch.zeros(len(lens), dtype=torch.int64, device=dev), None, None, layer, table,
                         lengths=lens)


def values_of(layer, table_row, n):
    """K and V (n, KVH, 64) in 64 bits of a row's first n slots."""
    state = row_state(layer, table_row, -(-n // 16) * 16)
    return [kv8.dense(*s)[:n] for s in state]


def check(got, want, v_max, what):
    off = np.abs(got.cpu().double().numpy() - want).max()
    assert off <= TOL * v_max, (what, off, TOL * v_max)


DECODE = [
    # rows' slots, kv heads, heads of each, page, pages a row
    ([1], 1, 1, 64, None),
    ([64], 2, 7, 64, None),
    ([65], 2, 7, 64, 40),
    ([1, 2, 15, 16, 17, 63, 64, 65, 127, 129], 2, 7, 64, None),
    ([1023, 0, 300, 4097], 2, 7, 64, None),
    ([5000], 1, 16, 64, 100),
    ([700, 3, 0, 1500, 200], 8, 2, 128, None),
    ([2000, 1111], 3, 5, 256, None),
    ([12345], 2, 8, 4096, None),
    ([33 * i % 500 for i in range(70)], 1, 4, 64, None),
]


def decode_case(gen, case, code, dev, size=1.0):
    rows, kvh, g, page, ppr = DECODE[case]
    ppr = ppr or max(1, -(-max(rows) // page))
    n_pages = sum(-(-n // page) for n in rows) + 3
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    table, host = make_table(gen, rows, page, n_pages, ppr, dev)
    fill_rows(gen, layer, table, rows, dev, size)
    q = torch.randn(len(rows), kvh, g, D, generator=gen).half().to(dev)
    last = torch.tensor([n - 1 for n in rows], dtype=torch.int64, device=dev)
    return rows, layer, table, host, q, last


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(dev, case, code):
    gen = torch.Generator().manual_seed(200 + case)
    rows, layer, table, host, q, last = decode_case(gen, case, code, dev)
    got = paged8.flash_decode_attention_paged8(q, layer, table, last)
    assert got.shape == q.shape
    for r, n in enumerate(rows):
        if n == 0:
            assert torch.equal(got[r], torch.zeros_like(got[r]))
            continue
        k, v = values_of(layer, host[r], n)
        want = kv8.attend(q[r].reshape(-1, D).cpu().double().numpy(), k, v)
        check(got[r].reshape(-1, D), want, np.abs(v).max(), (case, r, n))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("splits", [1, 3, 16, 40])
def test_split_phase_and_the_framework_s_merges(dev, code, splits):
    """Partials of any split count, merged by the merge of the fp16 caches."""
    gen = torch.Generator().manual_seed(31)
    rows, layer, table, host, q, last = decode_case(gen, 3, code, dev)
    b, kvh, g, _ = q.shape
    flash = ops.make_flash_scratch(b, kvh, g, table.shape[1] * 64, dev, splits=splits, fused=False)
    for t in flash[:3]:
        t.fill_(float("nan"))
    paged8.flash_decode_split_paged8(q, layer, table, flash, last)
    got = ops.flash_decode_combine(flash)
    for r, n in enumerate(rows):
        k, v = values_of(layer, host[r], n)
        want = kv8.attend(q[r].reshape(-1, D).cpu().double().numpy(), k, v)
        check(got[r].reshape(-1, D), want, np.abs(v).max(), (r, n))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_strided_queries_outputs_and_tables(dev, code):
    gen = torch.Generator().manual_seed(37)
    rows, layer, table, host, q, last = decode_case(gen, 4, code, dev)
    want = paged8.flash_decode_attention_paged8(q, layer, table, last, scale=0.3)
    b, kvh, g, _ = q.shape
    wide = torch.zeros(b, kvh, g + 2, 2 * D, device=dev, dtype=torch.float16)
    wide[:, :, 1:1 + g, D:] = q
    out = torch.full((b, g, kvh, D), 7.0, device=dev, dtype=torch.float16).transpose(1, 2)
    wide_table = torch.full((b, table.shape[1] + 3), -5, dtype=torch.int32, device=dev)
    wide_table[:, :table.shape[1]] = table
    lasts = torch.full((b, 3), 99, dtype=torch.int64, device=dev)
    lasts[:, 1] = last
    got = paged8.flash_decode_attention_paged8(wide[:, :, 1:1 + g, D:], layer, wide_table[:, :table.shape[1]],
                                               lasts[:, 1], scale=0.3, out=out)
    assert got is out and torch.equal(got, want)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_rows_do_not_depend_on_their_company(dev, code):
    """Nor on a row's place: the same rows in another order, bit for bit."""
    gen = torch.Generator().manual_seed(41)
    rows, layer, table, host, q, last = decode_case(gen, 4, code, dev)
    want = paged8.flash_decode_attention_paged8(q, layer, table, last)
    order = torch.tensor([3, 1, 0, 2], device=dev)
    got = paged8.flash_decode_attention_paged8(q[order], layer, table[order].contiguous(), last[order])
    assert torch.equal(got, want[order])
    parked = last.clone()
    parked[0] = parked[3] = -1
    got = paged8.flash_decode_attention_paged8(q, layer, table, parked)
    assert torch.equal(got[2], want[2]) and not got[0].any() and not got[3].any()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_unseen_slots_may_hold_anything(dev, code):
    """Slots behind the last one: NaN codes, NaN and infinite scales, in its block, tile and page."""
    for n in (1, 16, 20, 48, 63, 64, 100):
        gen = torch.Generator().manual_seed(43 + n)
        layer = tuple(t[0] for t in make_pools(gen, 4, 2, 64, code, dev, junk=False))
        table, host = make_table(gen, [128], 64, 4, 2, dev)
        fill_rows(gen, layer, table, [n], dev)
        q = torch.randn(1, 2, 7, D, generator=gen).half().to(dev)
        last = torch.tensor([n - 1], device=dev)
        want = paged8.flash_decode_attention_paged8(q, layer, table, last)
        for s in range(n, 128):
            page, off = int(host[0, s // 64]), s % 64
            layer[0].view(torch.uint8)[page, :, off] = 0x7F
            layer[1].view(torch.uint8)[page, :, 0, :, off] = 0xFF
            if s % 16 == 0:
                for t, x in zip(layer[2:], (float("nan"), float("inf")) if s % 32 else (-float("inf"), float("nan"))):
                    t[page, :, off // 16] = x
        assert torch.equal(paged8.flash_decode_attention_paged8(q, layer, table, last), want), n


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_nan_blocks_reach_who_sees_them(dev, code):
    gen = torch.Generator().manual_seed(47)
    layer = tuple(t[0] for t in make_pools(gen, 4, 2, 64, code, dev))
    table, host = make_table(gen, [200], 64, 4, 4, dev)
    fill_rows(gen, layer, table, [200], dev)
    q = torch.randn(1, 2, 7, D, generator=gen).half().to(dev)
    for which in (2, 3):
        keep = layer[which].clone()
        layer[which][int(host[0, 2]), 1, 1] = float("nan")            # slots 144 .. 159 of head 1
        seen = [paged8.flash_decode_attention_paged8(q, layer, table, torch.tensor([n - 1], device=dev))
                for n in (144, 145, 200)]
        assert torch.isfinite(seen[0]).all()
        for x in seen[1:]:
            assert torch.isnan(x[0, 1]).all() and torch.isfinite(x[0, 0]).all()
        layer[which].copy_(keep)


def test_scores_of_minus_infinity_alone(dev):
    """An infinite query against keys of the other sign: NaN, as from the fp16 caches."""
    for code in ("int8", "e4m3"):
        kv = paged8.PagedKv8Cache(1, 1, 2, 64, 1, 2, dev, code)
        kv.map_row(0, 100)
        x = torch.ones(100, 1, D, device=dev, dtype=torch.float16)
        cu = torch.tensor([0, 100], dtype=torch.int32, device=dev)
        paged8.append_paged8(-x, x, cu, 100, torch.zeros(1, dtype=torch.int64, device=dev), None, None,
                             kv.pools[0], kv.table)
        q = torch.ones(1, 1, 2, D, device=dev, dtype=torch.float16)
        q[0, 0, 1] = float("inf")
        got = paged8.flash_decode_attention_paged8(q, kv.pools[0], kv.table, torch.tensor([99], device=dev))
        assert torch.isnan(got[0, 0, 1]).all() and torch.equal(got[0, 0, 0], x[0, 0])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_values_of_very_different_sizes(dev, code):
    """Blocks whose scales lie far apart: a query that looks at the small ones gets them to their own precision."""
    gen = torch.Generator().manual_seed(53)
    kv = paged8.PagedKv8Cache(1, 1, 4, 64, 1, 4, dev, code)
    kv.map_row(0, 256)
    v = torch.randn(256, 1, D, generator=gen)
    size = torch.ones(256)
    size[:64], size[64:128], size[128:192], size[192:] = 6e4 / 5, 1.0, 2.0 ** -10, 2.0 ** -18
    v = (v.clamp(-5, 5) * size[:, None, None]).half()
    k = torch.zeros(256, 1, D)
    for j in range(4):
        k[64 * j:64 * j + 64, 0, j] = 8.0
    cu = torch.tensor([0, 256], dtype=torch.int32, device=dev)
    paged8.append_paged8(k.half().to(dev), v.to(dev), cu, 256, torch.zeros(1, dtype=torch.int64, device=dev), None,
                         None, kv.pools[0], kv.table)
    q = torch.zeros(1, 1, 4, D)
    for j in range(4):
        q[0, 0, j, j] = 64.0                          # 64 a score: the others' weight is e^-64
    got = paged8.flash_decode_attention_paged8(q.half().to(dev), kv.pools[0], kv.table,
                                               torch.tensor([255], device=dev))[0, 0]
    vals = values_of(kv.pools[0], kv.table[0].cpu(), 256)[1][:, 0]
    for j in range(4):
        part = vals[64 * j:64 * j + 64]
        off = np.abs(got[j].cpu().double().numpy() - part.mean(axis=0))
        # p are 1; the fp16 output's step below 2^-14 is 2^-24.
        assert (off <= TOL * np.abs(part).max() + 2.0 ** -25).all(), (j, off.max())


EXTEND = [
    # new tokens, slots before them, kv heads, heads of each, page
    ([1], [0], 1, 1, 64),
    ([5, 5], [300, 2011], 2, 7, 64),
    ([1, 8, 3], [15, 0, 64], 2, 7, 64),
    ([30], [100], 2, 7, 64),
    ([0, 17, 4, 2, 1], [5, 3, -1, 1000, 63], 8, 2, 128),
    ([70, 9, 130], [16, 1031, 0], 2, 7, 64),
    ([200], [700], 1, 16, 256),
    ([3] * 9, [100 * i for i in range(9)], 2, 8, 64),
    ([2], [5000], 1, 4, 64),
]


def extend_case(gen, case, code, dev):
    lens, ctx, kvh, g, page = EXTEND[case]
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // page) for n in need) + 3
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    table, host = make_table(gen, need, page, n_pages, max(1, -(-max(need) // page)), dev)
    fill_rows(gen, layer, table, ctx, dev)
    total = sum(lens)
    qkv = torch.randn(total, (g + 2) * kvh, D, generator=gen).half().to(dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    return (lens, ctx, kvh, g, layer, table, host, qkv[:, :g * kvh], qkv[:, g * kvh:(g + 1) * kvh],
            qkv[:, (g + 1) * kvh:], cu, torch.tensor(ctx, device=dev))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(EXTEND)))
def test_extend(dev, case, code):
    gen = torch.Generator().manual_seed(300 + case)
    lens, ctx, kvh, g, layer, table, host, q, k, v, cu, context = extend_case(gen, case, code, dev)
    other = tuple(t.clone() for t in layer)
    most = max(n + c for n, c in zip(lens, ctx))
    got = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), context, None, None, layer, table, lengths=lens,
                                       max_slots=most)
    paged8.append_paged8(k, v, cu, max(lens), context, None, None, other, table, lengths=lens)
    for a, b in zip(layer, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for r, (n, c) in enumerate(zip(lens, ctx)):
        lo = sum(lens[:r])
        if c < 0:
            assert not got[lo:lo + n].any()
            continue
        if n == 0:
            continue
        kk, vv = values_of(layer, host[r], c + n)
        for i in range(n):
            want = kv8.attend(q[lo + i].cpu().double().numpy(), kk[:c + i + 1], vv[:c + i + 1])
            check(got[lo + i], want, np.abs(vv).max(), (case, r, i))
    again = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), context, None, None, layer, table)
    assert torch.equal(again, got) or most < table.shape[1] * layer[0].shape[2]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_extend_rotates_queries_and_keys(dev, code):
    gen = torch.Generator().manual_seed(59)
    lens, ctx, kvh, g, layer, table, host, q, k, v, cu, context = extend_case(gen, 5, code, dev)
    n = q.shape[0]
    ang = torch.rand(n, 32, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], dim=1).half().to(dev) for f in (torch.cos, torch.sin))
    other = tuple(t.clone() for t in layer)
    got = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), context, cos, sin, layer, table, lengths=lens)

    def turn(x):
        cache = torch.zeros(n, kvh, 64, D, device=dev, dtype=torch.float16)
        y = ops.rope_append(x[:, :, None].contiguous(), k[:, :, None].contiguous(), v[:, :, None].contiguous(),
                            cos.view(n, 1, D), sin.view(n, 1, D), cache, cache.clone(),
                            torch.zeros(1, dtype=torch.int64, device=dev))
        return y[:, :, 0], cache[:, :, 0]

    q2, k2 = turn(q)
    want = paged8.prefill_extend_paged8(q2, k2, v, cu, max(lens), context, None, None, other, table, lengths=lens)
    assert torch.equal(got, want)
    for a, b in zip(layer, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_nan_tokens_reach_later_blocks_only(dev, code):
    """A token that is not finite: its block's queries and the later ones, not those of earlier blocks."""
    gen = torch.Generator().manual_seed(61)
    for which in (0, 1):
        layer = tuple(t[0] for t in make_pools(gen, 3, 1, 64, code, dev))
        table, host = make_table(gen, [90], 64, 3, 2, dev)
        fill_rows(gen, layer, table, [20], dev)
        x = torch.randn(2, 60, 1, D, generator=gen).half()
        x[which, 17, 0, 3] = float("nan")                              # slot 37, block 32 .. 47
        k, v = x.to(dev)
        q = torch.randn(60, 2, D, generator=gen).half().to(dev)
        cu = torch.tensor([0, 60], dtype=torch.int32, device=dev)
        got = paged8.prefill_extend_paged8(q, k, v, cu, 60, torch.tensor([20], device=dev), None, None, layer, table)
        assert torch.isfinite(got[:12]).all() and torch.isnan(got[12:]).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_max_slots_bounds_writes_and_reads(dev, code):
    gen = torch.Generator().manual_seed(67)
    layer = tuple(t[0] for t in make_pools(gen, 4, 1, 64, code, dev))
    table, host = make_table(gen, [200], 64, 4, 4, dev)
    fill_rows(gen, layer, table, [90], dev)
    x = torch.randn(30, 4, D, generator=gen).half().to(dev)
    cu = torch.tensor([0, 30], dtype=torch.int32, device=dev)
    ctx = torch.tensor([90], device=dev)
    other = tuple(t.clone() for t in layer)
    before = row_state(layer, host[0], 128)
    got = paged8.prefill_extend_paged8(x[:, :2], x[:, 2:3], x[:, 3:], cu, 30, ctx, None, None, layer, table,
                                       max_slots=100)
    for which, at in ((0, 2), (1, 3)):
        values, scales = before[which]
        kv8.append(values, scales, 90, x[:10, at:at + 1].cpu().double().numpy(), code)
        after = row_state(layer, host[0], 128)[which]
        assert np.array_equal(after[0], values) and np.array_equal(after[1], scales)
    kk, vv = values_of(layer, host[0], 100)
    for i in (0, 9, 10, 29):
        n = min(91 + i, 100)
        want = kv8.attend(x[i, :2].cpu().double().numpy(), kk[:n], vv[:n])
        check(got[i], want, np.abs(vv).max(), i)


# --------------------------------------------------------------------------
# a decoding step: the new token appended by the launch that attends
# --------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", [1, 2, 3, 4, 6, 8, 9])
def test_step_is_append_then_attend(dev, case, code):
    """Bit for bit, at every place in a block, parked rows left alone."""
    gen = torch.Generator().manual_seed(400 + case)
    rows, layer, table, host, q, last = decode_case(gen, case, code, dev)
    b, kvh, g, _ = q.shape
    other = tuple(t.clone() for t in layer)
    kv = (torch.randn(b, 3, kvh, D, generator=gen) * 2.0 ** torch.randint(-3, 4, (b, 1, 1, 1), generator=gen)).half()
    kv = kv.to(dev)
    key, value = kv[:, 0], kv[:, 2]
    cu = torch.arange(b + 1, dtype=torch.int32, device=dev)
    paged8.append_paged8(key, value, cu, 1, last, None, None, other, table)
    want = paged8.flash_decode_attention_paged8(q, other, table, last)
    got = paged8.flash_decode_attention_paged8(q, layer, table, last, key=key, value=value)
    assert torch.equal(got, want)
    for a, c in zip(layer, other):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    flash = ops.make_flash_scratch(b, kvh, g, table.shape[1] * layer[0].shape[2], dev, splits=5, fused=False)
    fresh = tuple(t.clone() for t in layer)
    paged8.flash_decode_split_paged8(q, fresh, table, flash, last, key=key * 3, value=value)
    paged8.append_paged8(key * 3, value, cu, 1, last, None, None, other, table)
    for a, c in zip(fresh, other):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))


def test_step_at_a_slot_without_a_page(dev):
    """Past the row's pages nothing is written and the row attends to all it has; an unmapped page is skipped."""
    gen = torch.Generator().manual_seed(71)
    layer = tuple(t[0] for t in make_pools(gen, 5, 2, 64, "int8", dev))
    table, host = make_table(gen, [128, 64], 64, 5, 2, dev)
    fill_rows(gen, layer, table, [128, 64], dev)
    before = tuple(t.clone() for t in layer)
    q = torch.randn(2, 2, 7, D, generator=gen).half().to(dev)
    new = torch.randn(2, 2, D, generator=gen).half().to(dev)
    got = paged8.flash_decode_attention_paged8(q, layer, table, torch.tensor([128, 70], device=dev), key=new, value=new)
    for a, c in zip(layer, before):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    want = paged8.flash_decode_attention_paged8(q, layer, table, torch.tensor([127, 70], device=dev))
    assert torch.equal(got[0], want[0])


# --------------------------------------------------------------------------
# graphs, streams, far pages
# --------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_captured_steps_replay(dev, code):
    """Two graphs over one cache, replayed in turn with eager calls between: each replay is the eager step's."""
    gen = torch.Generator().manual_seed(73)
    rows = [100, 0, 1100, 15]
    layer = tuple(t[0] for t in make_pools(gen, 60, 2, 64, code, dev))
    table, host = make_table(gen, [n + 40 for n in rows], 64, 60, 20, dev)
    fill_rows(gen, layer, table, rows, dev)
    mirror = tuple(t.clone() for t in layer)
    q = torch.zeros(4, 2, 7, D, device=dev, dtype=torch.float16)
    new = torch.zeros(2, 4, 2, D, device=dev, dtype=torch.float16)
    last = torch.tensor([n if n else -1 for n in rows], device=dev)
    cu = torch.arange(5, dtype=torch.int32, device=dev)

    def step(pools):
        return paged8.flash_decode_attention_paged8(q, pools, table, last, key=new[0], value=new[1])

    def long_step(pools):
        out = paged8.prefill_extend_paged8(q.view(4, 14, D), new[0], new[1], cu, 1, last, None, None, pools, table,
                                           lengths=[1, 1, 1, 1])
        return out, paged8.read_paged8(pools, table, cu, 1, last, lengths=[1, 1, 1, 1])

    graphs = []
    for fn in (step, long_step):
        pools = tuple(t.clone() for t in layer)
        fn(pools)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn(layer)
        graphs.append((g, out))
    for i in range(6):
        q.copy_(torch.randn(q.shape, generator=gen))
        new.copy_(torch.randn(new.shape, generator=gen))
        graphs[i % 2][0].replay()
        got = graphs[i % 2][1]
        torch.cuda.synchronize()
        want = (step, long_step)[i % 2](mirror)
        flat = lambda x: [x] if isinstance(x, torch.Tensor) else [x[0], *x[1]]  # noqa: E731
        for a, c in zip(flat(got), flat(want)):
            assert torch.equal(a, c), i
        for a, c in zip(layer, mirror):
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8)), i
        last += (last >= 0).long()


def test_two_streams_at_once(dev):
    """Calls on two streams over one cache: workspaces are each call's own."""
    gen = torch.Generator().manual_seed(79)
    rows, layer, table, host, q, last = decode_case(gen, 4, "int8", dev)
    qs = [torch.randn(q.shape, generator=gen).half().to(dev) for _ in range(8)]
    want = [paged8.flash_decode_attention_paged8(x, layer, table, last) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for i, x in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(paged8.flash_decode_attention_paged8(x, layer, table, last))
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert torch.equal(a, c)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_pages_past_four_gigabytes(dev, code):
    """A pool of 6 GB: pages whose offsets pass 32 bits are written, read and attended as the first ones are."""
    kvh, page, n_pages = 2, 256, 90000
    kv = paged8.PagedKv8Cache(1, kvh, n_pages, page, 2, 6, dev, code)
    gen = torch.Generator().manual_seed(83)
    far = [n_pages - 1, 70000, 66000, n_pages - 7, 69999]
    near = [0, 5, 2, 9, 1]
    n = 1111
    x = torch.randn(n, 4, D, generator=gen).half().to(dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    q = torch.randn(1, 2, 7, D, generator=gen).half().to(dev)
    got = []
    for r, pages in enumerate((near, far)):
        kv.table[r, :5] = torch.tensor(pages, dtype=torch.int32)
        t = kv.table[r:r + 1]
        paged8.append_paged8(x[:, :2], x[:, 2:], cu, n, zero, None, None, kv.pools[0], t)
        got.append((*paged8.read_paged8(kv.pools[0], t, cu, n, zero),
                    paged8.flash_decode_attention_paged8(q, kv.pools[0], t, torch.tensor([n - 1], device=dev))))
    for a, c in zip(*got):
        assert torch.equal(a, c)
    k, v = (t.double().cpu().numpy() for t in got[1][:2])
    check(got[1][2].reshape(-1, D), kv8.attend(q.reshape(-1, D).cpu().double().numpy(), k, v), np.abs(v).max(), "far")
    # Page copies over the same distance.
    paged8.copy_pages8(kv.store, far, [20, 21, 22, 23, 24])
    assert torch.equal(kv.store[0, 20:25], kv.store[0, far])


# --------------------------------------------------------------------------
# every form of the extension, past its loops' first rounds
# --------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh,g,cap", [
    ([700, 0, 513, 640], [0, 3, 100, 33], 4, 7, None),              # 128 query rows a workgroup, from an odd slot on
    ([400] * 6, [0, 64, 1, 15, 300, 17], 4, 8, None),
    ([129, 128, 127, 1], [0, 0, 0, 1], 64, 1, None),
    ([200], [5900], 16, 16, None),
    ([200], [12801], 8, 16, None),                                  # the same, cut along slots
    ([300, 250], [3000, 2500], 8, 7, None),                         # 48 query rows
    ([70], [2500], 2, 7, None),                                     # 32, in pieces
    ([2, 1], [4500, 4300], 1, 2, None),                             # 16, in pieces
    ([60], [10], 2, 7, 65536),                                      # a bound far above what is there
])
def test_extension_forms(dev, lens, ctx, kvh, g, cap, code):
    """Sampled queries of long rows: the first and last of each, those around block, tile and workgroup edges."""
    gen = torch.Generator().manual_seed(500 + lens[0] + kvh)
    page = 128
    need = [c + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // page) for n in need) + 1
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    ppr = -(-(cap or max(need)) // page)
    table, host = make_table(gen, need, page, n_pages, ppr, dev)
    fill_rows(gen, layer, table, ctx, dev)
    total = sum(lens)
    qkv = torch.randn(total, (g + 2) * kvh, D, generator=gen).half().to(dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    got = paged8.prefill_extend_paged8(qkv[:, :g * kvh], qkv[:, g * kvh:(g + 1) * kvh], qkv[:, (g + 1) * kvh:], cu,
                                       max(lens), torch.tensor(ctx, device=dev), None, None, layer, table, lengths=lens,
                                       max_slots=cap or max(need))
    assert torch.isfinite(got).all()
    for r, (n, c) in enumerate(zip(lens, ctx)):
        if n == 0:
            continue
        k, v = values_of(layer, host[r], c + n)
        edges = {0, 1, n - 1, n - 2, n // 2} | {128 // g * j + e for j in range(1, 9) for e in (-1, 0, 1)} \
            | {64 * j - c % 64 + e for j in range(1, 6) for e in (-1, 0)}
        for i in sorted(e for e in edges if 0 <= e < n):
            q = qkv[sum(lens[:r]) + i, :g * kvh].cpu().double().numpy()
            check(got[sum(lens[:r]) + i], kv8.attend(q, k[:c + i + 1], v[:c + i + 1]), np.abs(v).max(), (r, i))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_wide_extension_with_nan_blocks_and_junk(dev, code):
    """As the narrow form: NaN tokens reach their block's and later queries, slots behind the row hold anything."""
    gen = torch.Generator().manual_seed(89)
    kvh, n, c, b = 8, 300, 20, 6
    layer = tuple(t[0] for t in make_pools(gen, 40, kvh, 64, code, dev))
    table, host = make_table(gen, [n + c] * b, 64, 40, 6, dev)
    fill_rows(gen, layer, table, [c] * b, dev)
    # Behind the rows: NaN codes and scales.
    for r in range(b):
        page = int(host[r, (n + c) // 64])
        for t, x in ((layer[0], 0x7F), (layer[1], 0xFF)):
            t.view(torch.uint8)[page] = x
        for t in layer[2:]:
            t[page, :, (n + c) % 64 // 16 + 1:] = float("nan")
    x = torch.randn(2, b * n, kvh, D, generator=gen).half()
    x[0, 100, 1, 3] = float("nan")                    # row 0, slot 120 (block 112 .. 127), head 1: K
    x[1, 2 * n + 5, 2, 7] = float("inf")              # row 2, slot 25 (block 16 .. 31), head 2: V
    q = torch.randn(b * n, kvh * 7, D, generator=gen).half().to(dev)
    cu = torch.arange(0, (b + 1) * n, n, dtype=torch.int32, device=dev)
    ctx = torch.tensor([c, c, c, -1, c, c], device=dev)
    got = paged8.prefill_extend_paged8(q, x[0].to(dev), x[1].to(dev), cu, n, ctx, None, None, layer, table)
    bad = torch.isnan(got).view(b, n, kvh, 7 * D).all(-1).cpu()
    assert torch.equal(bad, ~torch.isfinite(got).view(b, n, kvh, 7 * D).all(-1).cpu())
    want = torch.zeros(b, n, kvh, dtype=torch.bool)
    want[0, 112 - c:, 1] = True
    want[2, 0:, 2] = True                             # slots 16 .. 19 of that block are older ones: all see it
    assert torch.equal(bad, want)
    assert not got[3 * n:4 * n].any()


def test_wild_device_arrays_stay_in_bounds(dev):
    """Offsets, slots, tables and contexts of any contents: nothing outside is touched, the call comes back, and rows
    that are right are right.  (Offsets can only be wrong where they are not read on the host: with ``lengths``.)"""
    gen = torch.Generator().manual_seed(97)
    for code in ("int8", "e4m3"):
        pools = make_pools(gen, 8, 2, 64, code, dev)
        layer = tuple(t[0] for t in pools)
        table, host = make_table(gen, [200, 150], 64, 8, 4, dev)
        fill_rows(gen, layer, table, [200, 150], dev)
        kv = torch.randn(9, 4, D, generator=gen).half().to(dev)
        q = torch.randn(9, 14, D, generator=gen).half().to(dev)
        lengths = [5, 4]
        big = [2 ** 63 - 1, 2 ** 40 + 5, 2 ** 31, 10 ** 6, -2 ** 63]
        for cu in ([0, 5, 9], [0, 9, 0], [7, 3, 20], [-4, 100, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 5]):
            cu = torch.tensor(cu, dtype=torch.int32, device=dev)
            for a in big + [100]:
                for wild in (table, torch.full_like(table, 2 ** 31 - 1), torch.full_like(table, -2 ** 31)):
                    ctx = torch.tensor([a, 100], device=dev)
                    work = tuple(t.clone() for t in layer)
                    paged8.append_paged8(kv[:, :2], kv[:, 2:], cu, 5, ctx, None, None, work, wild, lengths=lengths)
                    paged8.read_paged8(work, wild, cu, 5, ctx, lengths=lengths)
                    paged8.prefill_extend_paged8(q, kv[:, :2], kv[:, 2:], cu, 5, ctx, None, None, work, wild,
                                                 lengths=lengths)
                    g = q[:2].view(2, 2, 7, D)
                    paged8.flash_decode_attention_paged8(g, work, wild, ctx, key=kv[:2, :2], value=kv[:2, 2:])
                    torch.cuda.synchronize()
    cu = torch.tensor([0, 5, 9], dtype=torch.int32, device=dev)
    ctx = torch.tensor([2 ** 40, 100], device=dev)
    work = tuple(t.clone() for t in layer)
    got = paged8.prefill_extend_paged8(q, kv[:, :2], kv[:, 2:], cu, 5, ctx, None, None, work, table, lengths=lengths)
    k, v = values_of(work, host[1], 104)
    for i in range(4):
        check(got[5 + i], kv8.attend(q[5 + i].cpu().double().numpy(), k[:101 + i], v[:101 + i]), np.abs(v).max(), i)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh,g", [
    ([1, 2, 4, 3], [14, 15, 30, 2000], 2, 7),                       # appended by the attention's own launch
    ([32, 16, 1, 0, 31], [0, 1, 17, 5, 16], 3, 1),
    ([2, 1, 2], [100, -1, 63], 1, 16),
    ([6] * 70, [i * 9 % 400 for i in range(70)], 2, 7),             # 42 query rows, units enough
    ([33, 2], [40, 100], 2, 1),                                     # one query row more: by a launch of its own
])
def test_short_extensions_append_as_the_append_does(dev, lens, ctx, kvh, g, code):
    """Bit for bit in the pages, rotated keys too; the attention is over them."""
    gen = torch.Generator().manual_seed(700 + len(lens) + g)
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // 64) for n in need) + 2
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, 64, code, dev))
    table, host = make_table(gen, need, 64, n_pages, 32, dev)
    fill_rows(gen, layer, table, ctx, dev)
    total = sum(lens)
    qkv = spread(gen, total, (g + 2) * kvh, D).to(dev)
    q, k, v = qkv[:, :g * kvh], qkv[:, g * kvh:(g + 1) * kvh], qkv[:, (g + 1) * kvh:]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    ang = torch.rand(total, 32, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], dim=1).half().to(dev) for f in (torch.cos, torch.sin))
    context = torch.tensor(ctx, device=dev)
    for turn in ((None, None), (cos, sin)):
        a, c = tuple(t.clone() for t in layer), tuple(t.clone() for t in layer)
        paged8.append_paged8(k, v, cu, max(lens), context, *turn, a, table, lengths=lens)
        got = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), context, *turn, c, table, lengths=lens)
        for x, y in zip(a, c):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for r, (n, c0) in enumerate(zip(lens, ctx)):
        lo = sum(lens[:r])
        if c0 < 0:
            assert not got[lo:lo + n].any()
        elif n:
            kk, vv = values_of(c, host[r], c0 + n)
            state = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), context, None, None,
                                                 tuple(t.clone() for t in layer), table, lengths=lens)
            plain = tuple(t.clone() for t in layer)
            paged8.append_paged8(k, v, cu, max(lens), context, None, None, plain, table, lengths=lens)
            kk, vv = values_of(plain, host[r], c0 + n)
            for i in {0, n - 1}:
                want = kv8.attend(q[lo + i].cpu().double().numpy(), kk[:c0 + i + 1], vv[:c0 + i + 1])
                check(state[lo + i], want, np.abs(vv).max(), (r, i))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh", [
    ([150, 400, 0, 333], [64, 5, 7, 90], 8),                        # shared tiles
    ([600], [9000], 8),                                             # the same, in pieces that are joined
    ([20, 9], [2500, 2100], 2),                                     # the waves' own tiles, in pieces
])
def test_captured_chunks_replay(dev, lens, ctx, kvh, code):
    """A captured extension's replays, on a stream of its own, are the eager calls' on another, both running."""
    gen = torch.Generator().manual_seed(800 + kvh + len(lens))
    rounds = 3
    need = [c + rounds * n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // 64) for n in need) + 1
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, 64, code, dev))
    table, host = make_table(gen, need, 64, n_pages, -(-max(need) // 64), dev)
    fill_rows(gen, layer, table, ctx, dev)
    mirror = tuple(t.clone() for t in layer)
    total = sum(lens)
    qkv = torch.zeros(total, 9 * kvh, D, device=dev, dtype=torch.float16)
    at = torch.tensor(ctx, device=dev)
    step = torch.tensor(lens, device=dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)

    def chunk(x, pools, at):
        return paged8.prefill_extend_paged8(x[:, :7 * kvh], x[:, 7 * kvh:8 * kvh], x[:, 8 * kvh:], cu, max(lens), at, None,
                                            None, pools, table, lengths=lens, max_slots=max(need))

    chunk(qkv, tuple(t.clone() for t in layer), at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chunk(qkv, layer, at)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for i in range(rounds):
        x = torch.randn(qkv.shape, generator=gen).half().to(dev)
        qkv.copy_(x)
        here = at.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            want = chunk(x, mirror, here)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, c in zip(layer, mirror):
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8)), i
        at += step


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,ctx,kvh,g,cap", [
    ([300, 0, 250, 128], [6000, 3, 1000, 9000], 8, 7, None),
    ([300, 40, 250, 128], [6000, -1, 1000, 9000], 8, 7, None),      # a parked row inside the line
    ([6] * 70, [i * 9 % 400 for i in range(70)], 2, 16, 65536),     # more rows than lanes, little work for each
    ([300, 280], [700, 900], 8, 16, 1 << 23),                       # costs in coarser quanta
    ([1500], [7000], 2, 7, 1 << 15),
])
def test_extension_in_even_pieces(dev, lens, ctx, kvh, g, cap, code):
    """Pieces that begin and end inside units, that hold several, and none; as the definition, and as the rows one
    by one."""
    gen = torch.Generator().manual_seed(900 + len(lens) + kvh)
    page = 4096 if cap and cap > 1 << 20 else 128
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // page) for n in need) + 1
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    ppr = -(-(cap or max(need)) // page)
    table, host = make_table(gen, need, page, n_pages, ppr, dev)
    fill_rows(gen, layer, table, ctx, dev)
    total = sum(lens)
    qkv = torch.randn(total, (g + 2) * kvh, D, generator=gen).half().to(dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    q, k, v = qkv[:, :g * kvh], qkv[:, g * kvh:(g + 1) * kvh], qkv[:, (g + 1) * kvh:]
    got = paged8.prefill_extend_paged8(q, k, v, cu, max(lens), torch.tensor(ctx, device=dev), None, None, layer, table,
                                       lengths=lens, max_slots=cap or max(need))
    assert torch.isfinite(got).all()
    for r in range(0, len(lens), max(1, len(lens) // 8)):
        n, c, lo = lens[r], ctx[r], sum(lens[:r])
        if n == 0 or c < 0:
            assert not got[lo:lo + n].any()
            continue
        kk, vv = values_of(layer, host[r], c + n)
        edges = {0, 1, n - 1, n // 2} | {128 // g * j + e for j in range(1, 5) for e in (-1, 0, 1)}
        for i in sorted(e for e in edges if 0 <= e < n):
            check(got[lo + i], kv8.attend(qkv[lo + i, :g * kvh].cpu().double().numpy(), kk[:c + i + 1], vv[:c + i + 1]),
                  np.abs(vv).max(), (r, i))
        # Every token: the row by itself, whose units are cut elsewhere or not at all.
        alone = paged8.prefill_extend_paged8(q[lo:lo + n], k[lo:lo + n], v[lo:lo + n],
                                             torch.tensor([0, n], dtype=torch.int32, device=dev), n,
                                             torch.tensor([c], device=dev), None, None,
                                             tuple(t.clone() for t in layer), table[r:r + 1], max_slots=c + n)
        check(got[lo:lo + n], alone.cpu().double().numpy(), np.abs(vv).max(), r)


def test_wild_device_arrays_in_long_extensions(dev):
    """As for short ones: workgroups that find their work from such arrays come back, and touch nothing outside."""
    gen = torch.Generator().manual_seed(101)
    kvh, g, total = 8, 7, 600
    layer = tuple(t[0] for t in make_pools(gen, 90, kvh, 64, "int8", dev))
    table, host = make_table(gen, [2000, 1500, 700], 64, 90, 60, dev)
    fill_rows(gen, layer, table, [1800, 1200, 500], dev)
    x = torch.randn(total, (g + 2) * kvh, D, generator=gen).half().to(dev)
    q, k, v = x[:, :g * kvh], x[:, g * kvh:(g + 1) * kvh], x[:, (g + 1) * kvh:]
    for rows, most in ((3, 1024), (3, None), (2, None)):
        lengths = [total // rows] * rows
        for cu in ([0, 200, 400, 600], [0, 600, 0, 600], [500, 3, 20, -7], [-4, 100, 2 ** 31 - 1, 5],
                   [2 ** 31 - 1, -2 ** 31, 5, 600]):
            cu = torch.tensor(cu[:rows + 1], dtype=torch.int32, device=dev)
            for a in (2 ** 63 - 1, 2 ** 40 + 5, 2 ** 31, 10 ** 6, -2 ** 63, 100):
                ctx = torch.tensor([a, 100, a][:rows], device=dev)
                for wild in (table, torch.full_like(table, 2 ** 31 - 1)):
                    out = paged8.prefill_extend_paged8(q, k, v, cu, lengths[0], ctx, None, None,
                                                       tuple(t.clone() for t in layer), wild[:rows], lengths=lengths,
                                                       max_slots=most)
                    torch.cuda.synchronize()
                    assert out.shape == q.shape
    cu = torch.tensor([0, 200, 400, 600], dtype=torch.int32, device=dev)
    ctx = torch.tensor([2 ** 40, 1200, -5], device=dev)
    got = paged8.prefill_extend_paged8(q, k, v, cu, 200, ctx, None, None, layer, table, lengths=[200] * 3)
    kk, vv = values_of(layer, host[1], 1400)
    for i in (0, 1, 17, 18, 100, 198, 199):
        check(got[200 + i], kv8.attend(q[200 + i].cpu().double().numpy(), kk[:1201 + i], vv[:1201 + i]),
              np.abs(vv).max(), i)
    assert not got[400:].any()
