"""Lists of pages and rows hold whole numbers: nothing is cut to one (no GPU)."""

import numpy as np
import pytest
import torch

from qwenforge_amd import paged


def test_fractions_are_refused():
    kv = paged.PagedKvCache(layers=1, kv_heads=1, n_pages=4, page_size=64, max_rows=4, pages_per_row=2,
                            device="cpu")
    kv.map_row(0, 128)
    for rows in ([1.5], ["1"], [torch.tensor(1.0)]):
        with pytest.raises(TypeError):
            kv.fork_rows(0, rows, 64)
    kv.fork_rows(0, [np.int64(1), torch.tensor(2)], 64)
    assert kv.row_pages(1) == kv.row_pages(2) == [0]
    for pages in ([0.9], [None], np.array([1.0])):
        with pytest.raises(TypeError):
            paged._page_list("src", pages, 1, 0, 4)
    assert paged._page_list("src", np.array([3, 0]), 2, 0, 4) == [3, 0]
    assert paged._page_list("src", torch.tensor([2]), 1, 0, 4) == [2]
