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

    def call(pools=(16, 32), sp=8192, src=16, dst=16, n=1, pages=4, kvh=2, page=64, d=64):
        import ctypes as C
        arr = None if pools is None else (C.c_void_p * len(pools))(*pools)
        return lib.qf_copy_pages(arr, 0 if pools is None else len(pools), sp, 4096, 64, src, dst, None,
                                 n, pages, kvh, page, d, None)

    assert call(n=0) == 0                                # nothing to do, nothing launched
    assert call(d=128) == -2 and call(page=96) == -2 and call(pages=0) == -2
    assert call(pools=None) == -1 and call(pools=(16, None)) == -1 and call(pools=(16, 8)) == -1
    assert call(sp=8188) == -1 and call(src=None) == -1 and call(n=-1) == -1 and call(kvh=0) == -1
