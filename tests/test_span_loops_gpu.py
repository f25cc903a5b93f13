"""The loops of the span attention kernels (``include/qf_prefix.h``) past their
first fill: rings that wrap, waves that take several tiles, rows whose pages pass
one window of 64, in every form of unit.

The cases have so many query rows that the work is cut along the keys hardly or
not at all; each states the splits it is meant to have, read off the workspace
(264 bytes a partial).  K holds zeros and ones and a query is -1000 in one
dimension: a slot whose K has a one there scores -125 (weight 2^-180, nothing in
fp32), the others 0, so every weight is one or nothing.  V holds whole numbers up
to 3, so the sums are exact in fp32 whatever their order, and an output is its
quotient rounded twice in fp32 and once to fp16: relative 2^-11 + 2^-22.  A slot
lost, read twice or taken for another moves an output by far more: the sums are a
few hundred.
"""

import pytest
import torch

from qwenforge_amd import _lib, paged

pytestmark = pytest.mark.gpu
D, PART = 64, 264
TOL = 2.0 ** -11 + 2.0 ** -22


def _bits(gen, *shape):
    return torch.randint(0, 2, shape, generator=gen).half()


def _whole(gen, *shape):
    return torch.randint(-3, 4, shape, generator=gen).half()


def _queries(gen, *shape):
    dim = torch.randint(0, D, shape, generator=gen)
    return torch.zeros(*shape, D, dtype=torch.float16).scatter_(-1, dim[..., None], -1000.0), dim


def _expect(dims, k, v, limits):
    """dims, limits (n,): query i over slots [0, limits[i]) of k, v (slots, 64), whole numbers in fp32."""
    w = (k[:, dims].T == 0) & (torch.arange(k.shape[0]) < limits[:, None])
    none = ~w.any(dim=1)                                 # every visible slot alike
    w[none] = torch.arange(k.shape[0]) < limits[none][:, None]
    w = w.float()
    return (w @ v).double() / w.sum(dim=1, keepdim=True).double()


def _close(got, want, what):
    off = (got.double() - want).abs() - TOL * want.abs()
    assert off.max().item() <= 0, what


def _row(pool, pages, h, n):
    """(n, 64) fp32 of kv head h of a row's first n slots."""
    page = pool.shape[2]
    at = torch.arange(n)
    return pool[pages[at // page].long(), h, at % page].float()


EXTENDS = {
    # lens, contexts, qh, kvh, page, splits
    # 128 query rows a unit, one split: units of 1 to 11 tiles.
    "wide-all-counts": ([700], [0], 56, 8, 64, 1),
    "wide-all-counts-page-256": ([640, 61], [37, 129], 56, 8, 256, 1),
    # Two splits of some 5500 slots: 87 tiles, two windows of pages.
    "wide-windows": ([2048], [9000], 14, 2, 64, 2),
    # 64 query rows a unit.
    "single-all-counts": ([9] * 40, [16 * i for i in range(40)], 56, 8, 64, 1),
    "single-windows": ([8] * 64, [9000 - 31 * i for i in range(64)], 14, 2, 64, 2),
    # 16 query rows a unit: a wave takes up to 18 tiles.
    "narrow-windows": ([2] * 256, [4600 - 17 * i for i in range(256)], 14, 2, 64, 1),
    "narrow-few-tiles": ([2] * 256, [3 * i for i in range(256)], 14, 2, 64, 1),
}


@pytest.mark.parametrize("name", EXTENDS)
def test_extension_counts_every_slot_once(dev, name):
    lens, ctx, qh, kvh, page, splits = EXTENDS[name]
    gen = torch.Generator().manual_seed(sum(lens) + qh)
    b, total = len(lens), sum(lens)
    ppr = max(-(-(n + c) // page) for n, c in zip(lens, ctx))
    need = _lib.load().qf_prefill_extend_workspace(b, qh, kvh, total, ppr * page)
    assert max(1, need // (total * qh * PART)) == splits
    # Whole pages of cached slots may be shared; those that take new tokens are the row's own.
    common, own = 170, [-(-(n + c) // page) - c // page for n, c in zip(lens, ctx)]
    n_pages = common + sum(own)
    kp, vp = _bits(gen, n_pages, kvh, page, D), _whole(gen, n_pages, kvh, page, D)
    table = torch.randint(0, common, (b, ppr), generator=gen, dtype=torch.int32)
    at = common
    for r, (c, n) in enumerate(zip(ctx, own)):
        table[r, c // page:c // page + n] = torch.arange(at, at + n)
        at += n
    q, dims = _queries(gen, total, qh)
    k, v = _bits(gen, total, kvh, D), _whole(gen, total, kvh, D)
    starts = [sum(lens[:r]) for r in range(b + 1)]
    kd, vd = kp.to(dev), vp.to(dev)
    got = paged.prefill_extend_paged(q.to(dev), k.to(dev), v.to(dev),
                                     torch.tensor(starts, dtype=torch.int32, device=dev), max(lens),
                                     torch.tensor(ctx, device=dev), None, None, kd, vd, table.to(dev),
                                     lengths=lens).cpu()
    kp, vp, g = kd.cpu(), vd.cpu(), qh // kvh
    for r in range(b) if b <= 64 else list(range(0, b, 5)) + [b - 1]:
        n, c = lens[r], ctx[r]
        t = torch.arange(n)
        if n > 300:                                      # a sample, and both ends
            t = torch.cat([t[:70], t[-70:], torch.randperm(n, generator=gen)[:160]])
        for h in range(kvh):
            kr, vr = _row(kp, table[r], h, c + n), _row(vp, table[r], h, c + n)
            assert torch.equal(kr[c:], k[starts[r]:starts[r + 1], h].float())
            assert torch.equal(vr[c:], v[starts[r]:starts[r + 1], h].float())
            heads = slice(h * g, (h + 1) * g)
            want = _expect(dims[starts[r] + t, heads].reshape(-1), kr, vr, (c + t + 1).repeat_interleave(g))
            _close(got[starts[r] + t, heads].reshape(-1, D), want, (name, r, h))


DECODES = {
    # rows of a group, groups, prefix slots, kvh, own slots of row r, splits of both kinds together
    # 128 query rows a unit, one split: 79 tiles; narrow units of up to ten.
    "wide": (64, 8, 5000, 8, lambda r: 1 + 7 * (r % 91), 2),
    # 64 query rows, two splits of 4500 slots; one row's own slots pass a window.
    "single": (8, 64, 9000, 2, lambda r: 5000 if r == 77 else 1 + 5 * (r % 60), 3),
    # 16 query rows: a wave takes 20 tiles of a prefix.
    "narrow": (2, 128, 5000, 2, lambda r: 1 + 3 * r, 2),
}


@pytest.mark.parametrize("name", DECODES)
def test_prefix_decode_counts_every_slot_once(dev, name):
    rows, groups, longest, kvh, own_of, splits = DECODES[name]
    gen = torch.Generator().manual_seed(longest + rows)
    g, page, b = 7, 64, rows * groups
    plens = [longest - 13 * (i % 29) for i in range(groups)]
    lens = [plens[r // rows] + own_of(r) for r in range(b)]
    lens[3], lens[b - 2] = plens[0] // 2, 0              # ends within the prefix; parked
    ppr = -(-max(lens) // page)
    need = _lib.load().qf_decode_attn_prefix_workspace(b, kvh, g, groups, ppr * page)
    assert need // (b * kvh * g * PART) == splits
    n_pages = 300
    kp, vp = _bits(gen, n_pages, kvh, page, D), _whole(gen, n_pages, kvh, page, D)
    table = torch.randint(0, n_pages, (b, ppr), generator=gen, dtype=torch.int32)
    for i, p in enumerate(plens):
        # Shared pages, and the slots behind them in the partly filled one too: any row's will do.
        table[i * rows:(i + 1) * rows, :-(-p // page)] = table[i * rows, :-(-p // page)].clone()
    q, dims = _queries(gen, b, kvh, g)
    got = paged.flash_decode_attention_prefix_paged(
        q.to(dev), kp.to(dev), vp.to(dev), table.to(dev),
        torch.tensor([i * rows for i in range(groups + 1)], dtype=torch.int32, device=dev),
        torch.tensor(plens, dtype=torch.int32, device=dev), torch.tensor([n - 1 for n in lens], device=dev)).cpu()
    assert not got[b - 2].any()
    for r in [0, 1, 3, 77 % b, b - 1] + list(range(5, b, 19)):
        for h in range(kvh) if lens[r] else ():
            kr, vr = _row(kp, table[r], h, lens[r]), _row(vp, table[r], h, lens[r])
            want = _expect(dims[r, h], kr, vr, torch.full((g,), lens[r]))
            _close(got[r, h], want, (name, r, h))
