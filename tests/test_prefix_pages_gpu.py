"""Page copies and forked rows (``paged.copy_pages``, ``PagedKvCache.fork_rows``,
``own_slots``, ``compact``): exact, and nothing else is touched."""

import pytest
import torch

from qwenforge_amd import paged

pytestmark = pytest.mark.gpu


def _expect(store, src, dst, slots):
    want = store.clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        n = store.shape[-2] if slots is None else slots[i]
        want[..., b, :, :n, :] = store[..., a, :, :n, :]
    return want


@pytest.mark.parametrize("page,kvh,lead", [(64, 2, (24, 2)), (64, 1, (1,)), (256, 3, (5,)),
                                           (4096, 2, (2,)), (128, 8, (131,))])
@pytest.mark.parametrize("form", ["lists", "device"])
def test_copies_pages_exactly(dev, page, kvh, lead, form):
    gen = torch.Generator().manual_seed(page + kvh)
    n_pages = 9
    store = torch.randn(*lead, n_pages, kvh, page, 64, generator=gen).half().to(dev)
    perm = torch.randperm(n_pages, generator=gen).tolist()
    src, dst = perm[:3], perm[3:6]
    for slots in (None, [page, 1, 0], [page - 1, 37, page // 2 + 1]):
        want = _expect(store, src, dst, slots)
        args = (src, dst, slots)
        if form == "device":
            args = [None if x is None else torch.tensor(x, dtype=torch.int32, device=dev) for x in args]
        paged.copy_pages(store, args[0], args[1], slots=args[2])
        assert torch.equal(store, want), (page, slots)


def test_strided_pools_one_source_for_many_and_no_pairs(dev):
    gen = torch.Generator().manual_seed(1)
    # Heads innermost but the dims: (pages, slots, heads, 64) memory, and a pad between pages.
    base = torch.randn(2, 7, 64 * 3 + 2, 2, 64, generator=gen).half().to(dev)
    pools = [b[:, :64].transpose(1, 2) for b in base]
    want = base.clone()
    want[:, 2, :11], want[:, 5, :64], want[:, 6, :1] = base[:, 4, :11], base[:, 4, :64], base[:, 4, :1]
    paged.copy_pages(pools, [4, 4, 4], [2, 5, 6], slots=[11, 64, 1])
    assert torch.equal(base, want)
    paged.copy_pages(pools, [], [])
    assert torch.equal(base, want)


def test_bad_pages_and_counts_on_the_device_copy_nothing_or_the_page(dev):
    store = torch.randn(2, 6, 2, 64, 64, device=dev).half()
    i32 = dict(dtype=torch.int32, device=dev)
    want = _expect(store, [1, 0], [3, 2], [64, 0])
    src = torch.tensor([-1, 0, 6, 0, 1, 0, 2**31 - 1], **i32)
    dst = torch.tensor([2, 6, 3, -5, 3, 2, 4], **i32)
    slots = torch.tensor([64, 64, 64, 64, 1000, -3, 64], **i32)
    paged.copy_pages(store, src, dst, slots=slots)
    assert torch.equal(store, want)


def test_list_arguments_are_checked(dev):
    store = torch.zeros(2, 6, 2, 64, 64, device=dev, dtype=torch.float16)
    for src, dst, slots in (([0], [6], None), ([-1], [1], None), ([0, 1], [2, 2], None),
                            ([0, 1], [1, 2], None), ([0], [0], None), ([0], [1], [65]), ([0], [1], [-1]),
                            ([0, 1], [2], None), ([0], [1], [1, 2])):
        with pytest.raises(ValueError):
            paged.copy_pages(store, src, dst, slots=slots)
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        paged.copy_pages(store, one, [1])
    with pytest.raises(TypeError):
        paged.copy_pages(store, one, one.long())
    with pytest.raises(ValueError):
        paged.copy_pages(store, one, torch.zeros(2, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        paged.copy_pages([store[0], store[1][:5]], [0], [1])
    with pytest.raises(TypeError):
        paged.copy_pages(store.float(), [0], [1])


def test_captured_copy_follows_its_device_arguments(dev):
    store = torch.randn(3, 8, 2, 64, 64, device=dev).half()
    i32 = dict(dtype=torch.int32, device=dev)
    src, dst = torch.tensor([0, 1], **i32), torch.tensor([2, 3], **i32)
    slots = torch.tensor([64, 5], **i32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        paged.copy_pages(store, src, dst, slots=slots)
    for a, b, n in (([0, 1], [2, 3], [64, 5]), ([7, 2], [4, 5], [1, 64]), ([-1, 6], [0, 1], [64, 33])):
        store.normal_()
        want = _expect(store, [x for x in a if x >= 0], [y for x, y in zip(a, b) if x >= 0],
                       [k for x, k in zip(a, n) if x >= 0])
        for t, x in ((src, a), (dst, b), (slots, n)):
            t.copy_(torch.tensor(x, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(store, want)


def test_rows_fork_take_their_own_pages_and_are_compacted(dev):
    kv = paged.PagedKvCache(layers=3, kv_heads=2, n_pages=24, page_size=64, max_rows=6, pages_per_row=4,
                            device=dev)
    kv.map_row(5, 70)                                    # two pages that go again: holes for compact
    kv.map_row(0, 200)
    kv.release_row(5)
    kv.store.normal_()
    def rows(r, n):
        return [torch.cat(kv.gather(i, r, n)) for i in range(3)]

    def same(a, b):
        return all(torch.equal(x, y) for x, y in zip(a, b))

    whole = rows(0, 200)
    kv.fork_rows(0, [1, 3], 150)
    kv.fork_row(0, 4, 192)
    for r, n in ((1, 150), (3, 150), (4, 192)):
        assert same(rows(r, n), [w[:, :n] for w in whole])
    assert [kv.shared_pages(r) for r in (0, 1, 3, 4)] == [3, 2, 2, 3]
    kv.map_row(1, 256)
    # A row writes behind its fork, another into slots it shared: nobody else sees it.
    page, slot = kv.row_pages(1)[2], 150 % 64
    kv.store[:, :, page, :, slot:] = 7.0
    assert kv.own_slots(4, 60, 10) == 2                  # slots 60..69 lie in two shared pages
    for j in (0, 1):
        kv.store[:, :, kv.row_pages(4)[j]] = 9.0
    assert same(rows(0, 200), whole) and same(rows(3, 150), [w[:, :150] for w in whole])
    assert same(rows(1, 150), [w[:, :150] for w in whole])
    assert same([x[:, 128:] for x in rows(4, 192)], [w[:, 128:192] for w in whole])
    kv.release_row(0)
    before = {r: rows(r, n) for r, n in ((1, 256), (3, 150), (4, 192))}
    used = 24 - kv.free_pages()
    moved = kv.compact()
    assert moved > 0 and kv.free_pages() == 24 - used
    assert sorted({p for r in (1, 3, 4) for p in kv.row_pages(r)}) == list(range(used))
    for r, n in ((1, 256), (3, 150), (4, 192)):
        assert same(rows(r, n), before[r])
        pages = kv.row_pages(r)
        assert kv.table[r].tolist() == pages + [-1] * (4 - len(pages))
    assert kv.shared_pages(3) == 2
    assert kv.compact() == 0
    for r in (1, 3, 4):
        kv.release_row(r)
    assert kv.free_pages() == 24
