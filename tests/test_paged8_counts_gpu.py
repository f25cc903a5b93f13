"""Every slot of the caches held in 8 bits counts once: attention whose result shows a single slot left out, read
twice or taken for another, at lengths where random values average it away.

Counts.  K is zero, so a query weighs all that it sees alike.  V holds a one in the dimension that names the slot's
place in its tile (even kv heads) or its tile modulo 64 (odd ones), zeros elsewhere: an output is the number of seen
slots of that name over the number of seen slots.  Ones, zeros and weights are exact in every step and sums of them
in fp32, so an output is a quotient rounded twice in fp32 and once to fp16: relative 2^-11 + 2^-22.  A name has a
few hundred slots at most, so one more or less shows.

Keys.  K holds vectors of +-4 and a query is one of them: that slot scores 128 and no other more than 100 (checked),
2^-40 of its weight: nothing once a weight is rounded to fp16, and no change of the fp32 sums that an output in fp16
shows.  The output is the slot's value, bit for bit.
"""

import numpy as np
import pytest
import torch

from oracle import kv8
from qwenforge_amd import _lib, paged8
from test_paged8_gpu import make_pools, make_table

D = 64
TOL = 2.0 ** -11 + 2.0 ** -22
EVEN_PIECES = 2 * 768 * 128 * 264 + 768 * 32    # the workspace of an extension in even pieces


def names(first, n, kvh):
    """V of slots [first, first + n): (n, kvh, 64)."""
    s = torch.arange(first, first + n)
    v = torch.zeros(n, kvh, D)
    for h in range(kvh):
        v[torch.arange(n), h, s % 64 if h % 2 == 0 else s // 64 % 64] = 1.0
    return v


def shares(n, kvh):
    """The output over slots [0, m) for m = 0 .. n: (n + 1, kvh, 64) in 64 bits."""
    v = names(0, n, kvh).double()
    sums = torch.cat([torch.zeros(1, kvh, D, dtype=torch.float64), v.cumsum(dim=0)])
    return sums / torch.arange(n + 1).clamp(min=1).view(-1, 1, 1)


def differs(got, want):
    return bool(((got.double().cpu() - want).abs() > TOL * want).any())


def test_one_slot_more_or_less_shows():
    """The comparison refuses the definition's own result with a slot or a tile left out, read twice or moved."""
    n = 12345
    v = names(0, n, 2).double().numpy()
    q, k = np.ones((2, D)), np.zeros((n, 2, D))
    want = shares(n, 2)[n]

    def result(keep):
        return torch.tensor(kv8.attend(q, k[keep], v[keep])).half()

    every = np.arange(n)
    assert not differs(result(every), want)
    for s in (0, 5000, 12287, 12344):
        assert differs(result(np.delete(every, s)), want)
        assert differs(result(np.append(every, s)), want)
        assert differs(result(np.where(every == s, (s + 65) % n, every)), want)
    assert differs(result(np.delete(every, slice(6400, 6464))), want)
    assert differs(result(np.delete(every, slice(12288, 12345))), want)


def shared_row(gen, n, kvh, page, code, dev, keys=None, values=None):
    """Pools and the pages of a row of n slots, K zero or ``keys``, V names or ``values``."""
    n_pages = -(-n // page) + 2
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    table, _ = make_table(gen, [n], page, n_pages, -(-n // page), dev)
    k = torch.zeros(n, kvh, D) if keys is None else keys
    v = names(0, n, kvh) if values is None else values
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    paged8.append_paged8(k.half().to(dev), v.half().to(dev), cu, n, torch.zeros(1, dtype=torch.int64, device=dev), None,
                         None, layer, table, lengths=[n])
    return layer, table


DECODES = [
    # rows' lengths, kv heads, heads of each, page, splits of a row
    ([1024, 1023, 1, 64, 65, 0, 777, 960, 961], 2, 7, 64, 1),
    ([1000] * 60 + [513, 449], 3, 16, 128, 1),                      # four waves a row
    ([12345, 12288, 12289, 4096, 4097, 8200, 63, 0], 2, 8, 64, 32),
    ([16000, 15999, 8192, 8193, 4160, 1], 1, 5, 256, 63),
    ([16000 - 123 * (i % 130) for i in range(130)], 2, 2, 64, 2),   # halves of more than 64 pages
]


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode_counts_every_slot(dev, case, code):
    lens, kvh, g, page, splits = DECODES[case]
    gen = torch.Generator().manual_seed(10 + case)
    most = max(lens)
    layer, table = shared_row(gen, most, kvh, page, code, dev)
    b = len(lens)
    table = table.repeat(b, 1)
    need = _lib.load().qf_decode_attn_paged8_workspace(b, kvh, g, table.shape[1] * page)
    assert need == (0 if splits == 1 else b * kvh * g * splits * 264)
    q = torch.randn(b, kvh, g, D, generator=gen).half().to(dev)
    got = paged8.flash_decode_attention_paged8(q, layer, table, torch.tensor(lens, device=dev) - 1)
    want = shares(most, kvh)[torch.tensor(lens)]
    assert not differs(got, want[:, :, None].expand(-1, -1, g, -1))


EXTENDS = [
    # new tokens, slots before them, kv heads, heads of each, page, slots of the call, splits (0: even pieces)
    ([3, 1, 2], [0, 1000, 777], 2, 7, 64, 1024, 1),                 # appended by the attention
    ([5] * 40, [i * 13 % 900 for i in range(40)], 2, 7, 64, 1024, 1),
    ([5, 5], [300, 2011], 2, 7, 64, 2048, 1),                       # 16 query rows a unit
    ([2, 1], [9000, 4300], 1, 2, 64, 9088, 35),
    ([70], [9000], 2, 7, 64, 9088, 16),                             # 32
    ([300, 250], [3000, 2500], 8, 7, 64, 3328, 1),                  # 48
    ([700, 0, 513, 640], [0, 3, 100, 33], 4, 7, 64, 704, 1),        # 128, shared tiles
    ([200], [5000], 16, 16, 64, 5248, 1),
    ([300, 0, 250, 128], [6000, 3, 1000, 9000], 8, 7, 64, 9152, 0),
    ([1500], [16000], 2, 7, 64, 17536, 0),
    ([300, 280], [700, 900], 8, 16, 4096, 1 << 23, 0),              # costs in coarser quanta
]


def extension(case, code, dev, gen, keys=None, values=None):
    """The pools, tables and packed K and V of a case whose rows hold the same slots, new ones among them."""
    lens, ctx, kvh, g, page, cap, splits = EXTENDS[case]
    need = [c + n for c, n in zip(ctx, lens)]
    n_pages = sum(-(-n // page) for n in need) + 1
    layer = tuple(t[0] for t in make_pools(gen, n_pages, kvh, page, code, dev))
    table, _ = make_table(gen, need, page, n_pages, cap // page, dev)
    most = max(need)
    k = (torch.zeros(most, kvh, D) if keys is None else keys[:most]).half()
    v = (names(0, most, kvh) if values is None else values[:most]).half()

    def packed(t, spans):
        return torch.cat([t[a:b] for a, b in spans]).to(dev)

    def starts(n):
        return torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=dev)

    old = [(0, c) for c in ctx]
    if sum(ctx):
        paged8.append_paged8(packed(k, old), packed(v, old), starts(ctx), max(ctx),
                             torch.zeros(len(ctx), dtype=torch.int64, device=dev), None, None, layer, table, lengths=ctx)
    new = list(zip(ctx, need))
    used = _lib.load().qf_prefill_extend_paged8_workspace(len(lens), kvh * g, kvh, sum(lens), max(lens), cap)
    assert used == (EVEN_PIECES if splits == 0 else 0 if splits == 1 else sum(lens) * kvh * g * splits * 264)
    seen = torch.cat([torch.arange(a + 1, b + 1) for a, b in new])

    def run(q, **kw):
        return paged8.prefill_extend_paged8(q.half().to(dev), packed(k, new), packed(v, new), starts(lens), max(lens),
                                            torch.tensor(ctx, device=dev), None, None, layer, table, lengths=lens, **kw)

    return run, seen, (layer, table)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(EXTENDS)))
def test_extension_counts_every_slot(dev, case, code):
    """Every token's output, with the call's slots bounded and by the table's width."""
    lens, ctx, kvh, g, page, cap, _ = EXTENDS[case]
    gen = torch.Generator().manual_seed(30 + case)
    run, seen, _ = extension(case, code, dev, gen)
    most = int(seen.max())
    want = shares(most, kvh)[seen][:, :, None].expand(-1, -1, g, -1).reshape(len(seen), kvh * g, D)
    q = torch.randn(len(seen), kvh * g, D, generator=gen)
    assert not differs(run(q, max_slots=cap), want)
    assert not differs(run(q), want)
    assert not differs(run(q, max_slots=most), want)


def planted(gen, n, kvh):
    """Keys of +-4 and values of their own for n slots."""
    return (torch.randint(0, 2, (n, kvh, D), generator=gen) * 8 - 4).float(), torch.randn(n, kvh, D, generator=gen)


def apart(keys, slots, limits):
    """Whether no other visible slot comes near the one that a query asks for, in any kv head."""
    for h in range(keys.shape[1]):
        k = keys[:, h]
        for at in range(0, len(slots), 2048):
            s = k[slots[at:at + 2048]] @ k.T / 8
            s[torch.arange(len(k)) >= limits[at:at + 2048, None]] = 0.0
            s[torch.arange(len(s)), slots[at:at + 2048]] = 0.0
            if float(s.max()) > 100.0:
                return False
    return True


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("n,kvh,g,page", [(1000, 2, 7, 64), (5003, 2, 16, 64), (12000, 1, 16, 128)])
def test_decode_finds_every_key(dev, n, kvh, g, page, code):
    gen = torch.Generator().manual_seed(50 + n)
    keys, values = planted(gen, n, kvh)
    layer, table = shared_row(gen, n, kvh, page, code, dev, keys, values)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    held = paged8.read_paged8(layer, table, cu, n, torch.zeros(1, dtype=torch.int64, device=dev))[1]
    assert apart(keys, torch.arange(n), torch.full((n,), n))
    b = -(-n // (4 * g))
    for lo in range(0, n, b * g):
        slots = torch.arange(lo, lo + b * g).clamp(max=n - 1)
        q = keys[slots].view(b, g, kvh, D).transpose(1, 2).half().to(dev)
        got = paged8.flash_decode_attention_paged8(q, layer, table.repeat(b, 1), torch.full((b,), n - 1, device=dev))
        assert torch.equal(got.transpose(1, 2).reshape(b * g, kvh, D), held[slots.to(dev)]), lo


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(EXTENDS)))
def test_extension_finds_keys(dev, case, code):
    """Each query another slot of those that it sees, its own and its neighbours' among them."""
    lens, ctx, kvh, g, page, cap, _ = EXTENDS[case]
    gen = torch.Generator().manual_seed(70 + case)
    need = [c + n for c, n in zip(ctx, lens)]
    keys, values = planted(gen, max(need), kvh)
    run, seen, (layer, table) = extension(case, code, dev, gen, keys, values)
    limits = seen.repeat_interleave(g)
    slots = (torch.rand(len(limits), generator=gen) * limits).long().minimum(limits - 1)
    near = torch.arange(len(limits)) % 5 == 0
    slots[near] = (limits[near] - 1 - torch.arange(int(near.sum())) % 3).clamp(min=0)
    some = torch.arange(0, len(slots), max(1, len(slots) // 4096))
    assert apart(keys, slots[some], limits[some])
    q = keys[slots].view(len(seen), g, kvh, D).transpose(1, 2).reshape(len(seen), kvh * g, D)
    got = run(q, max_slots=cap).view(len(seen), kvh, g, D).transpose(1, 2).reshape(len(slots), kvh, D)
    # What the pages hold of each row now.
    cu = torch.tensor([sum(need[:i]) for i in range(len(need) + 1)], dtype=torch.int32, device=dev)
    held = paged8.read_paged8(layer, table, cu, max(need), torch.zeros(len(need), dtype=torch.int64, device=dev),
                              lengths=need)[1]
    base = torch.tensor([sum(need[:r]) for r, n in enumerate(lens) for _ in range(n * g)])
    assert torch.equal(got, held[(base + slots).to(dev)])
