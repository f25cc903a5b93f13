"""Caches held in 8 bits: appends, reads and page copies against the oracle.

Scales are powers of two and a code is the nearest one to a quotient that is
exact, so codes, scales and what is read back are compared bit for bit.
"""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import paged8
from qwenforge_amd.ops import rope_append

pytestmark = pytest.mark.gpu
D = 64


def make_pools(gen, n_pages, kvh, page, code, dev, layers=1, junk=True):
    """All layers' pools, every byte random where ``junk``: unused memory would show."""
    kv = paged8.PagedKv8Cache(layers, kvh, n_pages, page, 1, 1, dev, code)
    if junk:
        raw = torch.randint(0, 256, kv.store.shape, generator=gen, dtype=torch.uint8)
        kv.store.copy_(raw)
        for s in kv.all_pools[2:]:
            s.copy_(2.0 ** torch.randint(-9, 3, s.shape, generator=gen).float())
        for c in kv.all_pools[:2]:           # codes that no append makes: -128 and NaN
            b = c.view(torch.uint8)
            bad = b == 128 if code == "int8" else (b & 127) == 127
            b.masked_fill_(bad, 3)
    return kv.all_pools


def make_table(gen, rows, page, n_pages, ppr, dev):
    """Rows of mapped slots -> (table on the device, pages of each row)."""
    free = torch.randperm(n_pages, generator=gen).tolist()
    table = torch.full((len(rows), ppr), -1, dtype=torch.int32)
    for r, n in enumerate(rows):
        for j in range(-(-n // page)):
            table[r, j] = free.pop()
    return table.to(dev), table


def row_state(pools, table_row, slots):
    """(values, scales) in 64 bits of a row's first ``slots`` slots, as the oracle holds them."""
    k, v, ks, vs = (t.cpu() for t in pools)
    page = k.shape[2]
    s = torch.arange(slots)
    where, off = table_row[s // page].long(), s % page
    got = []
    for which, codes, scale in ((0, k, ks), (1, v, vs)):
        b = codes.view(torch.uint8)
        b = b[where, :, off] if which == 0 else b[where, :, off // 64, :, off % 64]
        got.append((b.contiguous().view(codes.dtype).double().numpy(),
                    scale[where[::16], :, off[::16] // 16].double().numpy()))
    return got


def spread(gen, *shape):
    """fp16 of sizes over many powers of two."""
    x = torch.randn(*shape, generator=gen)
    return (x * 2.0 ** torch.randint(-6, 4, shape[:-1] + (1,), generator=gen)).half()


CASES = [
    # tokens of each row, slots before them, kv heads, page
    ([1], [0], 2, 64),
    ([1], [777], 2, 64),
    ([1, 1, 1, 1], [15, 16, 17, 63], 1, 64),
    ([5, 0, 16, 33], [3, 40, 0, 64], 2, 64),
    ([17, 1, 200, 64], [31, 127, 5, 192], 3, 128),
    ([300], [0], 8, 256),
    ([70, 30, 1], [0, -1, 2], 2, 64),
    ([1] * 70, list(range(70)), 1, 64),
    ([3] * 20 + [0] * 50 + [40], list(range(71)), 2, 64),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append_is_the_definition(dev, case, code):
    lens, ctx, kvh, page = CASES[case]
    gen = torch.Generator().manual_seed(100 + case)
    total = sum(lens)
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    ppr = max(1, -(-max(need) // page))
    n_pages = sum(-(-n // page) for n in need) + 3
    pools = make_pools(gen, n_pages, kvh, page, code, dev)
    table, host = make_table(gen, need, page, n_pages, ppr, dev)
    layer = tuple(t[0] for t in pools)
    before = [row_state(layer, host[r], -(-n // 16) * 16) for r, n in enumerate(need)]
    untouched = [t.clone() for t in layer]
    # K and V as views of a fused projection's rows.
    qkv = spread(gen, total, 2 * kvh + 1, D).to(dev)
    k, v = qkv[:, 1:1 + kvh], qkv[:, 1 + kvh:]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    paged8.append_paged8(k, v, cu, max(lens), torch.tensor(ctx, device=dev), None, None, layer, table,
                         lengths=lens)
    for r, (n, c) in enumerate(zip(lens, ctx)):
        got = row_state(layer, host[r], -(-need[r] // 16) * 16)
        for which, new in ((0, k), (1, v)):
            values, scales = before[r][which]
            if c >= 0 and n:
                x = new[sum(lens[:r]):sum(lens[:r + 1])].cpu().double().numpy()
                kv8.append(values, scales, c, x, code)
            assert np.array_equal(got[which][1], scales), (r, which)
            assert np.array_equal(got[which][0], values), (r, which)
    # Pages of no row keep every byte.
    free = sorted(set(range(n_pages)) - set(host[host >= 0].tolist()))
    for t, u in zip(layer, untouched):
        assert torch.equal(t[free].view(torch.uint8), u[free].view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_tokens_one_by_one(dev, code):
    """A row filled token by token, growing: every step is the oracle's, and the first scale of a block
    forgets the page's last use."""
    gen = torch.Generator().manual_seed(7)
    layer = tuple(t[0] for t in make_pools(gen, 3, 2, 64, code, dev))
    table, host = make_table(gen, [80], 64, 3, 2, dev)
    x = (spread(gen, 80, 4, D) * torch.linspace(0.01, 3.0, 80)[:, None, None]).half()
    state = row_state(layer, host[0], 80)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    for i in range(80):
        t = x[i:i + 1].to(dev)
        paged8.append_paged8(t[:, :2], t[:, 2:], cu, 1, torch.tensor([i], device=dev), None, None, layer, table)
        for which in (0, 1):
            kv8.append(*state[which], i, x[i:i + 1, 2 * which:2 * which + 2].double().numpy(), code)
    got = row_state(layer, host[0], 80)
    for a, b in zip(got, state):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_every_half_rounds_to_its_code(dev, code):
    """All finite halves, in blocks of like size, as one block's largest and beside a larger one."""
    bits = torch.arange(0x7C00, dtype=torch.int32).to(torch.int16).view(torch.float16)
    n = bits.numel() // (D * 16) * D * 16
    for grown in (1.0, 60.0):
        x = bits[:n].view(-1, 1, D).clone()
        x[::2] *= -1
        if grown > 1:
            x[::16, 0, 0] = (x[::16, 0, 0].float().abs() * grown).clamp(max=65504.0).half()
        slots = x.shape[0]
        pages = -(-slots // 64)
        gen = torch.Generator().manual_seed(1)
        layer = tuple(t[0] for t in make_pools(gen, pages, 1, 64, code, dev))
        table, host = make_table(gen, [slots], 64, pages, pages, dev)
        cu = torch.tensor([0, slots], dtype=torch.int32, device=dev)
        zero = torch.zeros(1, dtype=torch.int64, device=dev)
        paged8.append_paged8(x.to(dev), x.flip(0).contiguous().to(dev), cu, slots, zero, None, None, layer, table)
        got = row_state(layer, host[0], slots)
        back = paged8.read_paged8(layer, table, cu, slots, zero)
        for which, y in ((0, x), (1, x.flip(0))):
            values, scales = np.zeros((slots, 1, D)), np.zeros((slots // 16, 1))
            kv8.append(values, scales, 0, y.double().numpy(), code)
            assert np.array_equal(got[which][1], scales)
            assert np.array_equal(got[which][0], values)
            assert np.array_equal(back[which].cpu().double().numpy(), kv8.dense(values, scales))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_every_code_at_every_scale_reads_exactly(dev, code):
    """Each code's value at each scale that fp16 holds it at, rounded to fp16.

    int8 values are exact: whole multiples of 2^-24.  So are all e4m3 values that an
    append writes -- fp16 inputs are multiples of 2^-24, and rounding one to a grid of
    a power of two leaves it on its own -- but at scales below 2^-15 there are e4m3
    codes between fp16's steps, which no append makes and which are read as the
    nearest of those."""
    lv = np.concatenate([kv8.levels(code), -kv8.levels(code)])
    exps = np.arange(-24, 11 if code == "int8" else 9)
    pages = -(-len(exps) // 4)
    kv = paged8.PagedKv8Cache(1, 1, pages, 64, 1, pages, dev, code)
    kv.map_row(0, pages * 64)
    codes = torch.tensor(lv).to(kv.pools[0][0].dtype).repeat(5)[:D * 16].view(16, D)
    k = codes.view(torch.uint8).repeat(pages * 4, 1).view(pages, 1, 64, D)
    for t, x in ((kv.pools[0][0], k), (kv.pools[0][1], k.transpose(2, 3).unsqueeze(2))):
        t.view(torch.uint8).copy_(x)
    s = torch.ones(pages * 4)
    s[:len(exps)] = torch.tensor(2.0 ** exps).float()
    for t in kv.pools[0][2:]:
        t.copy_(s.view(pages, 1, 4))
    got = kv.gather(0, 0, 64 * pages)
    want = codes.double().repeat(pages * 4, 1) * s.double().repeat_interleave(16)[:, None]
    want = want.where(want.abs() <= 65504, 0).half().double()
    for x in got:
        x = x[0].cpu().double()
        assert torch.equal(x.where(want != 0, 0), want)


def test_infinities_and_nan_make_a_block_nan(dev):
    for code in ("int8", "e4m3"):
        gen = torch.Generator().manual_seed(3)
        kv = paged8.PagedKv8Cache(1, 2, 4, 64, 1, 4, dev, code)
        kv.map_row(0, 200)
        table, layer = kv.table[:1], kv.pools[0]

        def put(x, at):
            x = x.to(dev)
            cu = torch.tensor([0, len(x)], dtype=torch.int32, device=dev)
            paged8.append_paged8(x[:, :2], x[:, 2:], cu, len(x), torch.tensor([at], device=dev), None, None,
                                 layer, table)

        x = torch.randn(100, 4, D, generator=gen).half()
        put(x, 0)
        clean = [t.clone() for t in kv.gather(0, 0, 100)]
        y = torch.randn(3, 4, D, generator=gen).half()
        y[1, 0, 5], y[2, 3, 63] = float("inf"), float("nan")
        put(y, 100)
        k, v = kv.gather(0, 0, 103)
        assert torch.isnan(k[0, 96:]).all() and torch.isnan(v[1, 96:]).all()
        for got, was, h in ((k, clean[0], 1), (v, clean[1], 0)):
            assert torch.isfinite(got[h]).all()
        assert torch.equal(k[:, :96], clean[0][:, :96]) and torch.equal(v[:, :96], clean[1][:, :96])
        put(x[:4], 103)                                   # the block stays NaN
        assert torch.isnan(kv.gather(0, 0, 107)[0][0, 96:]).all()
        put(x[:16], 96)                                   # and is itself again from its first slot on
        k, v = kv.gather(0, 0, 112)
        assert torch.isfinite(k).all() and torch.isfinite(v).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_rope_then_quantised(dev, code):
    """K rotated as rope_append rotates it."""
    gen = torch.Generator().manual_seed(5)
    n, kvh = 37, 2
    layer = tuple(t[0] for t in make_pools(gen, 3, kvh, 64, code, dev))
    other = tuple(t.clone() for t in layer)
    table, host = make_table(gen, [20 + n], 64, 3, 1, dev)
    kv = torch.randn(n, 2 * kvh, D, generator=gen).half().to(dev)
    ang = torch.rand(n, 32, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], dim=1).half().to(dev) for f in (torch.cos, torch.sin))
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    ctx = torch.tensor([20], device=dev)
    paged8.append_paged8(kv[:, :kvh], kv[:, kvh:], cu, n, ctx, cos, sin, layer, table)
    cache = torch.zeros(n, kvh, 64, D, device=dev, dtype=torch.float16)
    k4, v4 = kv[:, :kvh, None].contiguous(), kv[:, kvh:, None].contiguous()
    rope_append(k4, k4, v4, cos.view(n, 1, D), sin.view(n, 1, D), cache, cache.clone(),
                torch.zeros(1, dtype=torch.int64, device=dev))
    paged8.append_paged8(cache[:, :, 0], kv[:, kvh:], cu, n, ctx, None, None, other, table)
    for a, b in zip(layer, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_layers_at_once(dev, code):
    gen = torch.Generator().manual_seed(9)
    layers, kvh, n = 5, 2, 50
    pools = make_pools(gen, 4, kvh, 64, code, dev, layers=layers)
    one = [tuple(t[i].clone() for t in pools) for i in range(layers)]
    table, _ = make_table(gen, [60], 64, 4, 1, dev)
    k, v = (torch.randn(layers, n, kvh, D, generator=gen).half().to(dev) for _ in range(2))
    k = k.transpose(1, 2).contiguous().transpose(1, 2)            # heads outside tokens, as dense caches are
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    ctx = torch.tensor([7], device=dev)
    paged8.append_paged8(k, v, cu, n, ctx, None, None, pools, table)
    got = paged8.read_paged8(pools, table, cu, n, ctx)
    for i in range(layers):
        paged8.append_paged8(k[i], v[i], cu, n, ctx, None, None, one[i], table)
        for a, b in zip(pools, one[i]):
            assert torch.equal(a[i].view(torch.uint8), b.view(torch.uint8))
        for a, b in zip(got, paged8.read_paged8(one[i], table, cu, n, ctx)):
            assert torch.equal(a[i], b)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,longest", [(9, 1), (9, 37), (70, 1), (3, 700)])
def test_many_layers_at_once(dev, rows, longest, code):
    """More blocks than run at once, of new rows and of begun ones, with RoPE: as one layer at a time."""
    gen = torch.Generator().manual_seed(110 + rows + longest)
    layers, kvh, page = 24, 8, 64
    lens = [longest] + [max(1, longest - 5 * r) if longest > 1 else 1 for r in range(1, rows)]
    ctx = [[0, 5, 16, -1, 31, 77][r % 6] for r in range(rows)]
    need = [max(c, 0) + n for n, c in zip(lens, ctx)]
    n_pages = sum(-(-n // page) for n in need)
    pools = make_pools(gen, n_pages, kvh, page, code, dev, layers=layers)
    table, _ = make_table(gen, need, page, n_pages, -(-max(need) // page), dev)
    total = sum(lens)
    k, v = (spread(gen, layers, total, kvh, D).to(dev) for _ in range(2))
    ang = torch.rand(total, 32, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], dim=1).half().to(dev) for f in (torch.cos, torch.sin))
    cu = torch.tensor([sum(lens[:i]) for i in range(rows + 1)], dtype=torch.int32, device=dev)
    at = torch.tensor(ctx, device=dev)
    one = tuple(t.clone() for t in pools)
    paged8.append_paged8(k, v, cu, longest, at, cos, sin, pools, table, lengths=lens)
    for i in range(layers):
        paged8.append_paged8(k[i], v[i], cu, longest, at, cos, sin, tuple(t[i] for t in one), table, lengths=lens)
    for a, b in zip(pools, one):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_read_is_packed(dev, code):
    """Rows from the middle of blocks, empty, parked and past their pages."""
    gen = torch.Generator().manual_seed(11)
    kvh, page = 3, 128
    layer = tuple(t[0] for t in make_pools(gen, 9, kvh, page, code, dev))
    firsts, lens, mapped = [0, 130, 5, -1, 250, 77], [128, 0, 203, 9, 40, 1], [128, 256, 256, 256, 256, 128]
    table, host = make_table(gen, [128, 0, 256, 0, 256, 128], page, 9, 2, dev)
    first = torch.tensor(firsts, device=dev)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    total = starts[-1]
    cu = torch.tensor(starts, dtype=torch.int32, device=dev)
    for bad in (cu + 2, cu - 1, cu.flip(0)):
        with pytest.raises(ValueError, match="cu_seqlens"):
            paged8.read_paged8(layer, table, bad, max(lens), first, total=total)
    k, v = paged8.read_paged8(layer, table, cu, max(lens), first, total=total)
    assert k.shape == v.shape == (total, kvh, D)
    for r, (f, n) in enumerate(zip(firsts, lens)):
        state = row_state(layer, host[r].clamp(min=0), 256)
        for which, x in ((0, k), (1, v)):
            want = np.zeros((n, kvh, D))
            if f >= 0:
                have = kv8.dense(*state[which])[f:f + n]
                want[:len(have)] = have
            assert np.array_equal(x[starts[r]:starts[r + 1]].cpu().double().numpy(), want), (r, which)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_forked_rows_and_compaction(dev, code):
    gen = torch.Generator().manual_seed(13)
    kv = paged8.PagedKv8Cache(3, 2, 12, 64, 4, 3, dev, code)
    kv.map_row(0, 150)
    x = torch.randn(3, 150, 4, D, generator=gen).half().to(dev)
    cu = torch.tensor([0, 150], dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    paged8.append_paged8(x[:, :, :2], x[:, :, 2:], cu, 150, zero, None, None, kv.all_pools, kv.table[:1])
    want = [[t.clone() for t in kv.gather(i, 0, 150)] for i in range(3)]
    kv.fork_rows(0, [1, 3], 140)                             # the third page is copied
    assert kv.row_pages(1)[:2] == kv.row_pages(0)[:2] and kv.row_pages(1)[2] != kv.row_pages(0)[2]
    assert kv.own_slots(3, 0, 10) == 1
    kv.release_row(1)
    kv.release_row(0)
    kv.compact()
    for i in range(3):
        for a, b in zip(kv.gather(i, 3, 140), want[i]):
            assert torch.equal(a, b[:, :140])
    assert sorted(kv.row_pages(3)) == [0, 1, 2]


def test_refusals(dev):
    """Arguments that the calls refuse, each with one thing wrong."""
    kv = paged8.PagedKv8Cache(2, 2, 4, 64, 2, 2, dev, "int8")
    kv.map_row(0, 100)
    pools, table = kv.pools[0], kv.table
    x = torch.zeros(9, 2, D, device=dev, dtype=torch.float16)
    q = torch.zeros(9, 14, D, device=dev, dtype=torch.float16)
    g = torch.zeros(2, 2, 7, D, device=dev, dtype=torch.float16)
    cu = torch.tensor([0, 5, 9], dtype=torch.int32, device=dev)
    ctx = torch.zeros(2, dtype=torch.int64, device=dev)
    e4m3 = pools[0].view(torch.float8_e4m3fn)

    def append(key=x, value=x, cu=cu, longest=5, ctx=ctx, cos=None, sin=None, pools=pools, table=table, **kw):
        paged8.append_paged8(key, value, cu, longest, ctx, cos, sin, pools, table, **kw)

    def extend(query=q, key=x, value=x, cu=cu, longest=5, ctx=ctx, cos=None, sin=None, pools=pools, table=table, **kw):
        paged8.prefill_extend_paged8(query, key, value, cu, longest, ctx, cos, sin, pools, table, **kw)

    def read(pools=pools, table=table, cu=cu, longest=5, ctx=ctx, **kw):
        paged8.read_paged8(pools, table, cu, longest, ctx, **kw)

    def decode(grouped=g, pools=pools, table=table, ctx=ctx, **kw):
        paged8.flash_decode_attention_paged8(grouped, pools, table, ctx, **kw)

    k, v, ks, vs = pools
    bad_pools = [(k, v, ks), (k.float(), v, ks, vs), (k, v.view(torch.uint8), ks, vs), (k, v.view(torch.float8_e4m3fn), ks, vs),
                 (k, v, ks.half(), vs), (k, v.transpose(3, 4), ks, vs), (k, v, ks[:, :, :2], vs),
                 (k, v.contiguous(), ks, vs), (k, v, ks.contiguous(), vs), (k[..., :32], v, ks, vs), (k[:, :, :32], v, ks, vs),
                 (k, v, ks, vs.cpu()), (k[:0], v[:0], ks[:0], vs[:0]), kv.all_pools, (e4m3, v, ks, vs), None]
    for call in (append, extend, read, decode):
        for p in bad_pools:
            if call is read and p is kv.all_pools:
                continue
            with pytest.raises((TypeError, ValueError, RuntimeError)):
                call(pools=p)
        for t in (table.long(), table.cpu(), table[:1], table.t(), table[0], None):
            with pytest.raises((TypeError, ValueError)):
                call(table=t)
        for c in (ctx.int(), ctx.cpu(), ctx[:1], ctx.view(1, 2), None):
            with pytest.raises((TypeError, ValueError)):
                call(ctx=c)
    for call in (append, extend, read):
        for c in (cu.long(), cu.cpu(), cu[:1], cu.view(1, 3), cu + 1, cu.flip(0), cu.repeat_interleave(2)[::2], None):
            with pytest.raises((TypeError, ValueError)):
                call(cu=c)
        for n in (0, 4, 10):
            with pytest.raises(ValueError):
                call(longest=n)
        # (The read's total is the sum of lengths: 5 and 5 would be rows of another cu_seqlens.)
        for n in ([9], [5, 4, 0], [10, -1]) + (() if call is read else ([5, 5],)):
            with pytest.raises(ValueError):
                call(lengths=n)
    for call in (append, extend):
        for t in (x.float(), x.cpu(), x[..., :32], x[:, :1], x[:8], x[:, 0], x.transpose(0, 2), None):
            with pytest.raises((TypeError, ValueError, RuntimeError)):
                call(key=t)
            with pytest.raises((TypeError, ValueError, RuntimeError)):
                call(value=t)
        with pytest.raises(ValueError):
            call(cos=x[:, 0].contiguous())
        with pytest.raises(ValueError):
            call(cos=x[:8, 0].contiguous(), sin=x[:8, 0].contiguous())
        with pytest.raises((TypeError, RuntimeError)):
            call(cos=x[:, 0].float(), sin=x[:, 0].float())
    with pytest.raises(ValueError):
        append(key=x[None], value=x[None], pools=kv.all_pools)        # one layer's tokens, two layers' pools
    for t in (q.float(), q[:8], q[:, :13], q[:, :, :32], q[0], None):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            extend(query=t)
    with pytest.raises((ValueError, RuntimeError)):
        extend(query=torch.zeros(9, 34, D, device=dev, dtype=torch.float16))   # 17 heads of a kv head
    for n in (4, 129):
        with pytest.raises(ValueError):
            extend(max_slots=n)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan"))):
        for call in (extend, decode):
            with pytest.raises(RuntimeError, match="invalid"):
                call(**kw)
    for t in (g.float(), g[:1], g[:, :1], g[..., :32], g[0], None):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            decode(grouped=t)
    new = x[:2]
    for kw in (dict(out=g.float()), dict(out=g[:1]), dict(out=g.cpu()), dict(key=new), dict(value=new),
               dict(key=new, value=x[:1]), dict(key=new.float(), value=new), dict(key=new[:, :1], value=new[:, :1])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            decode(**kw)
    big = torch.zeros(200, 2, D, device=dev, dtype=torch.float16)
    with pytest.raises(ValueError, match="capacity"):
        append(key=big, value=big, cu=torch.tensor([0, 200, 200], dtype=torch.int32, device=dev), longest=200)
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([4], [0]), ([-1], [0]), ([0], [1, 2]), ([0.5], [1])):
        with pytest.raises((ValueError, TypeError)):
            paged8.copy_pages8(kv.store, src, dst)
    for store in (kv.store.view(torch.int8), kv.store[:, :2], kv.store[0], kv.store.cpu()):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            paged8.copy_pages8(store, [0], [1])
    for call in (append, extend, read, decode):
        call()                                                       # and as they are
