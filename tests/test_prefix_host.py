"""Host side of shared-prefix serving: page bookkeeping of forked rows and the
refusals of the entry points (no GPU)."""

import pytest
import torch

from qwenforge_amd import _lib, paged


def _cache(n_pages=12, max_rows=5, pages_per_row=4, **kw):
    return paged.PagedKvCache(layers=2, kv_heads=2, n_pages=n_pages, page_size=64, max_rows=max_rows,
                              pages_per_row=pages_per_row, device="cpu", **kw)


def test_forked_rows_share_whole_pages():
    kv = _cache()
    kv.map_row(0, 200)                                   # pages 0..3, the last partly filled
    kv.fork_rows(0, [2, 3], 128)                         # two whole pages: nothing to copy
    assert kv.row_pages(2) == kv.row_pages(3) == [0, 1]
    assert kv.table[2].tolist() == [0, 1, -1, -1]
    assert kv.free_pages() == 8 and kv.shared_pages(0) == 2
    assert kv.map_row(2, 130) == [0, 1, 4]
    kv.release_row(0)                                    # pages 2 and 3 were its own
    assert kv.free_pages() == 9 and kv.shared_pages(2) == 2
    assert kv.map_row(1, 64) == [2]
    kv.release_row(2)
    assert kv.row_pages(3) == [0, 1] and kv.shared_pages(3) == 0
    kv.release_row(3)
    assert kv.free_pages() == 11
    kv.release_row(3)                                    # nothing mapped: nothing happens
    assert kv.free_pages() == 11
    kv.fork_row(1, 4, 0)                                 # no slots: an empty row
    assert kv.row_pages(4) == [] and kv.table[4].tolist() == [-1] * 4


def test_refused_forks_leave_the_cache_as_it_was():
    kv = _cache(n_pages=5)
    kv.map_row(0, 200)
    before = (kv.free_pages(), kv.table.clone(), kv.row_pages(0))
    for rows, n in (([1], 257), ([1], -1), ([1, 1], 64), ([0], 64), ([5], 64), ([-1], 64)):
        with pytest.raises(ValueError):
            kv.fork_rows(0, rows, n)
    with pytest.raises(RuntimeError, match="exhausted"):
        kv.fork_rows(0, [1, 2], 100)                     # two partly filled pages, one free
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.fork_row(0, 1, 100)                           # a page to copy, but no GPU
    for first, n in ((0, 257), (-1, 3), (250, 10), (0, -1)):
        with pytest.raises(ValueError):
            kv.own_slots(0, first, n)
    assert (kv.free_pages(), kv.row_pages(0)) == (before[0], before[2])
    assert torch.equal(kv.table, before[1])


def test_own_slots_and_compact_without_anything_to_copy():
    kv = _cache()
    kv.map_row(0, 200)
    assert kv.own_slots(0, 0, 200) == 0 and kv.own_slots(0, 64, 0) == 0
    kv.fork_row(0, 1, 128)
    assert kv.own_slots(0, 128, 72) == 0                 # only the first two pages are shared
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.own_slots(1, 127, 1)
    assert kv.row_pages(1) == [0, 1] and kv.free_pages() == 8
    assert kv.compact() == 0


def test_copy_pages_refusals():
    pool = torch.zeros(4, 2, 64, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged.copy_pages(pool, [0], [1])
    with pytest.raises(ValueError):
        paged.copy_pages([], [0], [1])
    with pytest.raises(ValueError):
        paged.copy_pages(pool.transpose(0, 1), [0], [1])
    lib = _lib.load()

    def call(pools=(16, 32), sp=8192, src=16, dst=16, n=1, pages=4, kvh=2, page=64, d=64, per=1, step=8):
        import ctypes as C
        arr = None if pools is None else (C.c_void_p * len(pools))(*pools)
        return lib.qf_copy_pages(arr, 0 if pools is None else len(pools), per, step, sp, 4096, 64, src, dst, None,
                                 n, pages, kvh, page, d, None)

    assert call(n=0) == 0                                # nothing to do, nothing launched
    assert call(d=128) == -2 and call(page=96) == -2 and call(pages=0) == -2
    assert call(pools=None) == -1 and call(pools=(16, None)) == -1 and call(pools=(16, 8)) == -1
    assert call(sp=8188) == -1 and call(src=None) == -1 and call(n=-1) == -1 and call(kvh=0) == -1
    assert call(per=0) == -1 and call(per=65536) == -1 and call(step=4) == -1


def test_verify_refusals_without_a_gpu():
    from qwenforge_amd import verify

    lib = _lib.load()

    def call(logits=16, dtype=0, sn=100, tokens=16, au=16, su=16, q=None, qsn=100, temp=1.0, width=2, ws=16,
             bytes_=1 << 20, t=4, b=2, v=100):
        return lib.qf_verify_drafts(logits, dtype, sn, tokens, 16, au, su, q, qsn, temp, 16, width, 16, ws,
                                    bytes_, t, b, v, None)

    assert call(dtype=2) == -2 and call(t=0) == -1 and call(v=0) == -1 and call(b=0) == -1
    assert call(v=2**31 - 1, sn=2**31) == -2
    assert call(logits=None) == -1 and call(logits=17) == -1 and call(logits=18, dtype=1) == -1
    assert call(sn=99) == -1 and call(tokens=None) == -1 and call(au=None) == -1 and call(su=None) == -1
    assert call(q=16, qsn=99) == -1 and call(width=0) == -1 and call(ws=8) == -1
    assert call(temp=-0.5) == -1 and call(temp=float("nan")) == -1 and call(temp=float("inf")) == -1
    assert call(temp=1e-320) == -1 and call(temp=1e39) == -1 and call(temp=1e-39) == -1
    assert call(bytes_=8) == -3
    assert lib.qf_verify_workspace(4, 2, 100) > 0
    with pytest.raises(RuntimeError, match="no CPU path"):
        verify.verify_drafts(torch.zeros(2, 8), None, None, 1, None, None)


def test_span_attention_refusals_without_a_gpu():
    lib = _lib.load()

    def prefix(q=16, page=64, rows=16, plen=16, last=16, ws=16, bytes_=1 << 30, out=16, b=2, kvh=2, g=7, d=64,
               scale=0.125, q_sb=896, sn=64, groups=1, bt_sb=4, ppr=4, pt=None, pt_sb=4, ppp=4):
        return lib.qf_decode_attn_prefix_paged(q, q_sb, 448, 64, 16, 8192, 4096, sn, 16, 8192, 4096, 64, 16, bt_sb,
                                               ppr, 8, page, rows, plen, groups, pt, pt_sb, ppp, last, 1, ws,
                                               bytes_, out, 896, 448, 64, b, kvh, g, d, scale, None)

    assert prefix(d=128) == -2 and prefix(g=17) == -2 and prefix(page=32) == -2 and prefix(sn=56) == -2
    for bad in (dict(q=None), dict(q=8), dict(rows=None), dict(plen=None), dict(last=None), dict(ws=None),
                dict(ws=8), dict(out=None), dict(out=4), dict(b=0), dict(kvh=0), dict(groups=0), dict(q_sb=4),
                dict(bt_sb=3), dict(pt=16, ppp=0), dict(pt=16, pt_sb=3), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert prefix(**bad) == -1, bad
    assert prefix(bytes_=100) == -3
    assert lib.qf_decode_attn_prefix_workspace(0, 2, 7, 1, 64) == -1
    assert lib.qf_decode_attn_prefix_workspace(1, 2, 17, 1, 64) == -2
    assert prefix(groups=2**31 - 1) == -2
    assert lib.qf_decode_attn_prefix_workspace(1, 2, 7, 2**31 - 1, 64) == -2
    assert lib.qf_prefill_extend_workspace(2**31 - 1, 14, 2, 1, 64) == -2

    def extend(q=16, cu=16, total=8, ctx=16, cos=None, sin=None, cap=256, ws=16, bytes_=1 << 30, out=16, b=2,
               qh=14, kvh=2, d=64, k_sn=1152, ppr=4):
        return lib.qf_prefill_extend_paged(q, 64, 1152, 16, 64, k_sn, 16, 64, 1152, cu, total, ctx, 1, cos, sin, 64,
                                           16, 8192, 4096, 64, 16, 8192, 4096, 64, 16, 4, ppr, 8, 64, cap, ws,
                                           bytes_, out, 64, 896, b, qh, kvh, d, 0.125, None)

    assert extend(d=32) == -2 and extend(qh=34) == -2 and extend(ppr=0) == -2
    for bad in (dict(q=None), dict(cu=None), dict(total=0), dict(ctx=None), dict(cos=16), dict(sin=16),
                dict(cos=8, sin=16), dict(cap=0), dict(cap=257), dict(ws=None), dict(out=None), dict(b=0),
                dict(qh=13), dict(kvh=0), dict(k_sn=1150)):
        assert extend(**bad) == -1, bad
    assert extend(bytes_=16) == -3
    assert lib.qf_prefill_extend_workspace(2, 14, 2, 0, 256) == -1
