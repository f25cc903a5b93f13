"""Host side of the caches held in 8 bits: layout, page bookkeeping and the refusals of the
entry points (no GPU)."""

import ctypes
import struct

import pytest
import torch

from qwenforge_amd import _lib, paged8


def _cache(code="int8", **kw):
    args = dict(layers=2, kv_heads=2, n_pages=6, page_size=128, max_rows=4, pages_per_row=3, device="cpu")
    return paged8.PagedKv8Cache(**{**args, **kw}, code=code)


@pytest.mark.parametrize("code,dtype", [("int8", torch.int8), ("e4m3", torch.float8_e4m3fn)])
def test_pools_are_views_of_one_record_a_page(code, dtype):
    kv = _cache(code)
    assert kv.store.shape == (2, 6, 2 * 128 * 257 // 2) and kv.capacity == 384
    for i, (k, v, ks, vs) in enumerate(kv.pools):
        assert k.shape == (6, 2, 128, 64) and v.shape == (6, 2, 2, 64, 64) and ks.shape == vs.shape == (6, 2, 8)
        assert k.dtype is v.dtype is dtype and ks.dtype is vs.dtype is torch.float32
        for t, whole in zip((k, v, ks, vs), kv.all_pools):
            assert t.untyped_storage().data_ptr() == kv.store.untyped_storage().data_ptr()
            assert t.data_ptr() == whole[i].data_ptr() and t.stride() == whole[i].stride()
        # Records do not overlap and fill the store.
        kv.store.zero_()
        for n, t in enumerate((k, v)):
            t.view(torch.uint8).fill_(n + 1)
        ks.fill_(1.0)
        vs.fill_(1.0)
        per = kv.store[i].reshape(6, -1)
        assert (per == 1).sum() == 6 * 2 * 128 * 64 and (per == 2).sum() == 6 * 2 * 128 * 64
        assert (per == 0x3F).sum() == (per == 0x80).sum() == 2 * 6 * 2 * 8


def test_rows_and_pages_are_the_parent_s():
    kv = _cache()
    kv.map_row(0, 300)
    kv.fork_rows(0, [1], 256)
    assert kv.row_pages(1) == [0, 1] and kv.shared_pages(0) == 2
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.fork_rows(0, [2], 300)                        # a page to copy, but no GPU
    with pytest.raises(ValueError, match="code must be"):
        _cache("fp8")
    with pytest.raises(ValueError, match="page_size"):
        _cache(page_size=96)


def test_there_is_no_cpu_path():
    kv = _cache()
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: paged8.append_paged8(x, x, cu, 3, ctx, None, None, kv.pools[0], kv.table[:1]),
                 lambda: paged8.read_paged8(kv.pools[0], kv.table[:1], cu, 3, ctx),
                 lambda: paged8.flash_decode_attention_paged8(x[:1, None], kv.pools[0], kv.table[:1], ctx),
                 lambda: paged8.prefill_extend_paged8(x, x, x, cu, 3, ctx, None, None, kv.pools[0], kv.table[:1]),
                 lambda: paged8.copy_pages8(kv.store, [0], [1])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


# The structs of the C ABI with plausible values: addresses that are never followed, as
# every call here is refused before a launch.
POOL = dict(k=256, v=256, k_scale=256, v_scale=256, sl=0, sp=16448, sh=4096, ssl=0, ssp=16, ssh=4, table=256, bt_sb=4,
            pages_per_row=4, n_pages=8, page_size=64, layers=1, KVH=2, code=0)
ROWS = dict(POOL, tk=256, k_sl=0, k_sh=64, k_sn=128, tv=256, v_sl=0, v_sh=64, v_sn=128, cu=256, total=9, max_seqlen=5,
            first=256, first_sb=1, cos=0, sin=0, cs_sn=0, B=3, D=64)
DECODE = dict(POOL, q=256, q_sb=896, q_sh=448, q_sg=64, kv_last=256, kv_last_sb=1, out=256, o_sb=896, o_sh=448, o_sg=64,
              ws=256, ws_bytes=1 << 20, B=3, G=7, D=64, k_new=0, kn_sb=0, kn_sh=0, v_new=0, vn_sb=0, vn_sh=0, scale=0.125)
EXTEND = dict(ROWS, q=256, q_sh=64, q_sn=896, out=256, o_sh=64, o_sn=896, cap=256, ws=256, ws_bytes=1 << 24, QH=14,
              scale=0.125)


def _pack(fields):
    values = list(fields.values())
    return struct.pack("=%dq" % len(values), *values) if "scale" not in fields else \
        struct.pack("=%dqd" % (len(values) - 1), *values)


@pytest.mark.parametrize("change", [
    dict(k=0), dict(v_scale=0), dict(table=0), dict(k=264), dict(k_scale=258), dict(sp=16440), dict(bt_sb=3),
    dict(KVH=0), dict(layers=0), dict(code=2), dict(page_size=96), dict(page_size=32), dict(page_size=8192),
    dict(n_pages=0), dict(pages_per_row=0), dict(pages_per_row=1 << 31), dict(sh=-16),
    dict(D=128), dict(B=0), dict(total=0), dict(max_seqlen=0), dict(max_seqlen=10), dict(cu=0), dict(first=0),
    dict(tk=0), dict(tv=260), dict(k_sn=100), dict(B=1 << 31), dict(total=1 << 31, max_seqlen=1),
    dict(layers=70000), dict(KVH=40000, layers=2)])
def test_rows_are_refused_before_a_launch(change):
    lib = _lib.load()
    for name in ("qf_append_paged8", "qf_read_paged8"):
        assert getattr(lib, name)(_pack({**ROWS, **change}), None) in (-1, -2), name


@pytest.mark.parametrize("change", [dict(cos=256), dict(sin=256), dict(cos=256, sin=264, cs_sn=64),
                                    dict(cos=256, sin=256, cs_sn=60)])
def test_rope_tables_are_refused_before_a_launch(change):
    lib = _lib.load()
    assert lib.qf_append_paged8(_pack({**ROWS, **change}), None) == -1
    assert lib.qf_read_paged8(_pack({**ROWS, "cos": 256, "sin": 256, "cs_sn": 64}), None) == -1


@pytest.mark.parametrize("change", [
    dict(q=0), dict(q=264), dict(q_sg=60), dict(kv_last=0), dict(out=0), dict(out=260), dict(o_sg=62), dict(G=0),
    dict(G=17), dict(D=32), dict(B=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(layers=2),
    dict(k_new=256), dict(v_new=256), dict(k_new=256, v_new=264), dict(k_new=256, v_new=256, kn_sb=60), dict(n_pages=0),
    dict(B=1 << 40)])
def test_decode_is_refused_before_a_launch(change):
    lib = _lib.load()
    args = _pack({**DECODE, **change})
    assert lib.qf_decode_attn_paged8(args, None) in (-1, -2)
    if "out" not in change and "o_sg" not in change:
        assert lib.qf_decode_split_paged8(args, 256, 256, 256, 4, None) in (-1, -2)


def test_partials_are_refused_before_a_launch():
    lib = _lib.load()
    for acc, m, l, splits in ((0, 256, 256, 4), (264, 256, 256, 4), (256, 0, 256, 4), (256, 256, 0, 4),
                              (256, 256, 256, 0), (256, 256, 256, 2000)):
        assert lib.qf_decode_split_paged8(_pack(DECODE), acc, m, l, splits, None) == -1
    long = {**DECODE, "pages_per_row": 4096, "bt_sb": 4096}
    need = lib.qf_decode_attn_paged8_workspace(3, 2, 7, 4096 * 64)
    assert need > 0
    assert lib.qf_decode_attn_paged8(_pack({**long, "ws_bytes": need - 1}), None) == -3
    assert lib.qf_decode_attn_paged8(_pack({**long, "ws": 0}), None) == -1
    assert lib.qf_decode_attn_paged8_workspace(3, 2, 7, 1024) == 0      # in one piece
    for sizes in ((0, 2, 7, 64), (3, 0, 7, 64), (3, 2, 0, 64), (3, 2, 17, 64), (3, 2, 7, 0)):
        assert lib.qf_decode_attn_paged8_workspace(*sizes) < 0


@pytest.mark.parametrize("change", [
    dict(QH=13), dict(QH=0), dict(QH=64), dict(q=0), dict(q_sh=60), dict(out=0), dict(o_sn=62), dict(cap=0),
    dict(cap=257), dict(scale=0.0), dict(layers=2), dict(total=0), dict(max_seqlen=0), dict(max_seqlen=10), dict(cu=0),
    dict(first=0), dict(tk=0), dict(cos=256), dict(D=128), dict(k=0), dict(B=0)])
def test_extension_is_refused_before_a_launch(change):
    assert _lib.load().qf_prefill_extend_paged8(_pack({**EXTEND, **change}), None) in (-1, -2)


def test_extension_s_workspace():
    lib = _lib.load()
    for sizes in ((0, 14, 2, 9, 5, 256), (3, 13, 2, 9, 5, 256), (3, 14, 0, 9, 5, 256), (3, 14, 2, 0, 5, 256),
                  (3, 14, 2, 9, 0, 256), (3, 14, 2, 9, 5, 0), (3, 64, 2, 9, 5, 256)):
        assert lib.qf_prefill_extend_paged8_workspace(*sizes) < 0
    need = lib.qf_prefill_extend_paged8_workspace(3, 14, 2, 9, 5, 1 << 16)
    big = {**EXTEND, "pages_per_row": 1024, "bt_sb": 1024, "cap": 1 << 16, "ws_bytes": need - 1}
    assert need > 0 and lib.qf_prefill_extend_paged8(_pack(big), None) == -3


def test_copies_are_refused_before_a_launch():
    lib = _lib.load()
    good = dict(store=256, layers=2, layer_step=1600, step=160, bytes=160, src=256, dst=256, n=1, n_pages=10)
    for change in (dict(store=0), dict(store=264), dict(layers=0), dict(layer_step=1608), dict(step=152), dict(step=144),
                   dict(bytes=0), dict(bytes=152), dict(src=0), dict(dst=0), dict(n=-1), dict(n_pages=0),
                   dict(layers=70000)):
        assert lib.qf_copy_pages8(*{**good, **change}.values(), None) in (-1, -2), change
    assert lib.qf_copy_pages8(*{**good, "n": 0, "src": 0, "dst": 0}.values(), None) == 0
    assert ctypes.sizeof(ctypes.c_void_p) == 8
