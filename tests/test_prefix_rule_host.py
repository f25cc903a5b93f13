"""When ``serve`` reads a common prefix once for all rows: the cases that were
timed at more than one layout of heads, on the side that was faster (no GPU).  Cases
within the timing's noise (half a microsecond of some 30 a layer) say nothing."""

from types import SimpleNamespace

import pytest

from qwenforge_amd.paged_engine import PagedDecodeEngine

# heads, kv heads, rows, slots, us per layer alone, together
TIMED = [
    (14, 2, 2, 1024, 25.1, 27.4), (14, 2, 2, 4096, 30.6, 28.9), (14, 2, 2, 8192, 38.0, 30.9),
    (14, 2, 3, 2048, 27.7, 30.1), (14, 2, 3, 6144, 35.3, 31.6), (14, 2, 4, 2048, 28.6, 30.7),
    (14, 2, 4, 6144, 35.5, 32.7), (14, 2, 5, 8192, 32.2, 35.8), (14, 2, 5, 16384, 35.3, 37.0),
    (14, 2, 5, 32768, 41.6, 39.6), (14, 2, 8, 8192, 33.2, 38.0), (14, 2, 8, 16384, 36.6, 38.8),
    (14, 2, 8, 32768, 43.9, 40.0), (14, 2, 16, 8192, 39.3, 41.4), (14, 2, 16, 16384, 46.1, 43.5),
    (14, 2, 32, 4096, 45.4, 46.5), (14, 2, 32, 8192, 52.2, 48.0), (14, 2, 48, 2048, 89.2, 91.3),
    (14, 2, 48, 4096, 96.6, 91.5),
    (16, 8, 2, 2048, 28.2, 29.7), (16, 8, 2, 8192, 39.1, 36.6), (16, 8, 3, 6144, 36.1, 33.6),
    (16, 8, 4, 4096, 33.0, 35.7), (16, 8, 4, 8192, 40.5, 37.4), (16, 8, 5, 8192, 39.2, 38.6),
    (16, 8, 8, 4096, 37.2, 38.6), (16, 8, 8, 8192, 44.2, 40.9), (16, 8, 16, 4096, 47.6, 42.0),
    (16, 8, 32, 2048, 52.1, 47.6), (16, 8, 48, 2048, 114.1, 96.9),
    (16, 4, 2, 4096, 31.4, 29.8), (16, 4, 4, 2048, 29.4, 30.5), (16, 4, 4, 6144, 36.9, 32.7),
    (16, 4, 5, 8192, 35.0, 36.0), (16, 4, 5, 16384, 39.8, 38.0), (16, 4, 8, 8192, 37.5, 38.6),
    (16, 4, 8, 16384, 44.5, 41.7), (16, 4, 16, 8192, 47.8, 44.4), (16, 4, 32, 2048, 46.3, 47.7),
    (16, 4, 32, 4096, 53.3, 47.9),
    (8, 1, 2, 4096, 29.2, 26.5), (8, 1, 4, 2048, 26.4, 27.8), (8, 1, 4, 6144, 33.6, 29.0),
    (8, 1, 5, 32768, 33.4, 36.9), (8, 1, 8, 32768, 34.7, 38.1), (8, 1, 16, 16384, 36.6, 39.8),
    (8, 1, 32, 8192, 42.0, 43.9), (8, 1, 32, 16384, 48.8, 46.1), (8, 1, 48, 4096, 74.4, 75.3),
]


@pytest.mark.parametrize("heads,kv_heads,batch,slots,alone,once", TIMED)
def test_the_faster_side_is_taken(heads, kv_heads, batch, slots, alone, once):
    engine = SimpleNamespace(cfg=SimpleNamespace(heads=heads, kv_heads=kv_heads),
                             uses_fused_step=lambda rows: rows <= 4)
    assert PagedDecodeEngine.reads_prefix_once(engine, batch, slots) == (once < alone)


@pytest.mark.parametrize("fused", [True, False])
def test_a_row_alone_shares_with_nobody(fused):
    engine = SimpleNamespace(cfg=SimpleNamespace(kv_heads=8), uses_fused_step=lambda rows: fused)
    assert not PagedDecodeEngine.reads_prefix_once(engine, 1, 1 << 20)
