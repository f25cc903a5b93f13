"""Paged KV caches held in 8 bits (``include/qf_paged8.h``).

The reference keeps its caches in fp16 (SE:705-716).  Here a page of a kv head
holds int8 or e4m3 codes with a scale, a power of two, for each block of 16 slots:
half the bytes that a decoding step reads, and twice the slots in a GPU's memory.
A code's value, code * scale, is exact in fp16.

A layer's ``pools`` are ``(k, v, k_scale, v_scale)``:

* k (n_pages, KVH, P, 64): slot s of the page is ``k[page, h, s]``;
* v (n_pages, KVH, P / 64, 64, 64): its value is ``v[page, h, s // 64, :, s % 64]``
  (the dims of 64 slots side by side, as the matrix cores take them);
* k_scale, v_scale (n_pages, KVH, P / 16) fp32: of slot s ``[page, h, s // 16]``.

k and v are int8 (codes -127 .. 127) or float8_e4m3fn.  int8 keeps a block's values
to 1/254 .. 1/127 of its largest magnitude, e4m3 each to 1/16 of itself, also
where a few channels are far larger than the others.

* ``PagedKv8Cache`` -- ``paged.PagedKvCache`` over such pools.
* ``append_paged8`` -- new tokens quantised into their pages, with RoPE if asked.
* ``read_paged8`` -- slots of rows back in fp16.
* ``flash_decode_attention_paged8`` / ``flash_decode_split_paged8`` -- attention of
  single tokens (SE:834-874 semantics).
* ``prefill_extend_paged8`` -- new tokens appended and attended with the slots before
  them.
* ``copy_pages8`` -- pages of every layer copied to other pages in one launch.
"""

from __future__ import annotations

import torch

from . import _lib, paged
from .ops import HEAD_DIM, _ptr, _scratch_args
from .paged import _call, _check_page_size, _check_rows, _half, _int_rows, _page_list, _workspace

BLOCK = 16
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_KINDS = {torch.int8: 0, torch.float8_e4m3fn: 1}


class PagedKv8Cache(paged.PagedKvCache):
    """``PagedKvCache`` held in 8 bits: ``code`` is ``"int8"`` or ``"e4m3"``.

    ``pools[i]`` is layer i's ``(k, v, k_scale, v_scale)``, ``all_pools`` the same
    with the layers as a first dimension; both are views of ``store`` (layers,
    n_pages, bytes) uint8, which holds each page of a layer as one record.
    Rows, pages, forks, ``own_slots`` and ``compact`` are the parent's.
    """

    def __init__(self, layers: int, kv_heads: int, n_pages: int, page_size: int, max_rows: int,
                 pages_per_row: int, device, code: str = "int8"):
        if code not in CODES:
            raise ValueError(f"code must be one of {sorted(CODES)} (got {code!r})")
        self.code = code
        super().__init__(layers, kv_heads, n_pages, page_size, max_rows, pages_per_row, device,
                         CODES[code])

    def _allocate(self, layers: int, dtype) -> None:
        n, kvh, page = self.n_pages, self.kv_heads, self.page_size
        per, scales = kvh * page * HEAD_DIM, 4 * kvh * page // BLOCK
        store = torch.zeros((layers, n, 2 * (per + scales)), device=self.device, dtype=torch.uint8)
        k, v, ks, vs = store.split([per, per, scales, scales], dim=2)
        # What no token was written to reads as zero at a scale that is one.
        ks.view(torch.float32).fill_(2.0 ** -24)
        vs.view(torch.float32).fill_(2.0 ** -24)
        self.store = store
        self.all_pools = (k.view(dtype).unflatten(2, (kvh, page, HEAD_DIM)),
                          v.view(dtype).unflatten(2, (kvh, page // 64, HEAD_DIM, 64)),
                          ks.view(torch.float32).unflatten(2, (kvh, page // BLOCK)),
                          vs.view(torch.float32).unflatten(2, (kvh, page // BLOCK)))
        self.pools = list(zip(*self.all_pools))

    def _copy(self, src, dst, slots=None) -> None:
        # Whole pages: the slots behind a row's last are nobody's.
        copy_pages8(self.store, src, dst)

    def gather(self, layer: int, row: int, length: int):
        """Slots ``[0, length)`` of ``row`` as dense ``(KVH, length, 64)`` K and V."""
        if length < 1:
            empty = torch.empty((self.kv_heads, 0, HEAD_DIM), device=self.device, dtype=torch.float16)
            return empty, empty.clone()
        cu = torch.tensor([0, length], device=self.device, dtype=torch.int32)
        first = torch.zeros(1, device=self.device, dtype=torch.int64)
        k, v = read_paged8(self.pools[layer], self.table[row:row + 1], cu, length, first, lengths=[length])
        return k.transpose(0, 1), v.transpose(0, 1)


# --------------------------------------------------------------------------
# argument helpers
# --------------------------------------------------------------------------

def _pools8(pools, block_table, batch: int, index: int, layers: int = 0):
    """The ``Pool8`` of a layer's pools -- with ``layers``, of ``layers`` layers' as
    ``PagedKv8Cache.all_pools`` -- and the rows' table on GPU ``index``, and the slots
    of a row."""
    if not isinstance(pools, (tuple, list)) or len(pools) != 4:
        raise TypeError("pools must be (k, v, k_scale, v_scale)")
    k, v, ks, vs = pools
    for name, t in (("k", k), ("v", v), ("k_scale", ks), ("v_scale", vs)):
        if not isinstance(t, torch.Tensor) or t.get_device() != index or index < 0:
            raise RuntimeError(f"{name} must be a tensor on cuda:{index}; there is no CPU path")
    kind = _KINDS.get(k.dtype)
    if kind is None or v.dtype is not k.dtype or ks.dtype is not torch.float32 or vs.dtype is not torch.float32:
        raise TypeError("k and v must both be int8 or float8_e4m3fn, k_scale and v_scale float32 "
                        f"(got {k.dtype}, {v.dtype}, {ks.dtype}, {vs.dtype})")
    lead = 1 if layers else 0
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 + lead or (layers and shape[0] != layers):
        raise ValueError(f"k must be {'(layers, ' if layers else '('}n_pages, KVH, P, 64) (got {tuple(shape)})")
    n_pages, kvh, page, d = shape[lead:]
    _check_page_size(page)
    if (d != HEAD_DIM or n_pages < 1 or kvh < 1
            or v.shape != (*shape[:lead + 2], page // 64, HEAD_DIM, 64)
            or ks.shape != (*shape[:lead + 2], page // BLOCK) or vs.shape != ks.shape):
        raise ValueError(f"pools of {n_pages} pages of {kvh} heads and {page} slots need v (n_pages, KVH, "
                         f"P / 64, 64, 64) and scales (n_pages, KVH, P / {BLOCK})")
    scale_strides = ks.stride()
    outer, scale_outer = strides[:lead + 2], scale_strides[:lead + 2]
    if (v.stride() != (*outer, 4096, 64, 1) or strides[lead + 2:] != (64, 1)
            or vs.stride() != scale_strides or scale_strides[-1] != 1):
        raise ValueError("k and v must have the same page and head strides, and so must the scales; "
                         "what a page and head holds must be contiguous")
    if (not isinstance(block_table, torch.Tensor) or block_table.dtype is not torch.int32
            or block_table.get_device() != index):
        raise TypeError(f"block_table must be an int32 tensor on cuda:{index}")
    if block_table.dim() != 2 or block_table.shape[0] != batch or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be (B={batch}, pages_per_row) with unit inner stride")
    ppr = block_table.shape[1]
    if lead == 0:
        outer, scale_outer = (0, *outer), (0, *scale_outer)
    return _lib.Pool8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *outer, *scale_outer,
                      block_table.data_ptr(), block_table.stride(0), ppr, n_pages, page, layers or 1, kvh,
                      kind), ppr * page


def _packed(cu_seqlens, total: int, max_seqlen: int, first, name: str, index: int, lengths):
    """Rows of packed tokens and each one's first slot: their number and first's stride."""
    b = cu_seqlens.shape[0] - 1 if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.dim() == 1 else 0
    if b < 1 or not 1 <= max_seqlen <= total:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    if _int_rows("cu_seqlens", cu_seqlens, b + 1, torch.int32, index) != 1:
        raise ValueError("cu_seqlens must be contiguous")
    stride = _int_rows(name, first, b, torch.int64, index)
    _check_rows(cu_seqlens, total, max_seqlen, lengths)
    return b, stride


def _rope(cos, sin, total: int, index: int):
    """(cos, sin, token stride) of per-token tables (T, 64), or Nones."""
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is None:
        return None, None, 0
    for n, t in (("cos", cos), ("sin", sin)):
        _half(n, t, 2)
        if t.shape[0] != total or t.get_device() != index:
            raise ValueError(f"{n} must be (T={total}, 64) on cuda:{index}")
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin, cos.stride(0)


# --------------------------------------------------------------------------
# writing, reading, copying
# --------------------------------------------------------------------------

def append_paged8(key: torch.Tensor, value: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                  context: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None, pools,
                  block_table: torch.Tensor, lengths=None) -> None:
    """New tokens quantised into their pages: row b's token i goes to its slot
    context[b] + i.

    Packed key and value (T, KVH, 64) fp16; ``cu_seqlens`` (B + 1,) int32,
    ``max_seqlen`` and ``lengths`` as in ``paged.prefill_extend_paged`` (a row may
    have no tokens); ``context`` (B,) int64 is read on the device, and a row with a
    negative one (parked) appends nothing.  ``cos``/``sin`` (T, 64): key is rotated
    before it is quantised.  With key and value (layers, T, KVH, 64) and the pools of
    as many layers (``PagedKv8Cache.all_pools``), all layers' tokens at once.

    A block's scale is the least power of two, 2^-24 or more, at which the largest
    magnitude written to it since its first slot fits; tokens that need a larger one
    than the block has round the codes already there to it.  So what a block holds may
    depend on the calls that filled it, by half a step of its scale for each time
    that grew.  Tokens with infinities or NaN make their blocks read as NaN until
    the first slot is written again.  Pages written to must be the row's own.
    """
    layers = key.shape[0] if isinstance(key, torch.Tensor) and key.dim() == 4 else 0
    lead = 1 if layers else 0
    _half("key", key, 3 + lead)
    _half("value", value, 3 + lead)
    index = key.get_device()
    shape = key.shape
    total, kvh = shape[lead], shape[lead + 1]
    if value.shape != shape or value.get_device() != index:
        raise ValueError(f"key and value must be alike (got {tuple(shape)}, {tuple(value.shape)})")
    b, ctx_sb = _packed(cu_seqlens, total, max_seqlen, context, "context", index, lengths)
    pool, cap = _pools8(pools, block_table, b, index, layers)
    if pool.KVH != kvh:
        raise ValueError(f"pools hold {pool.KVH} kv heads, key {kvh}")
    if max_seqlen > cap:
        raise ValueError(f"max_seqlen exceeds the row capacity {cap}")
    cos, sin, cs_sn = _rope(cos, sin, total, index)
    ks, vs = key.stride(), value.stride()
    _call("qf_append_paged8", index, key.data_ptr(), ks[0] if layers else 0, ks[lead + 1], ks[lead],
          value.data_ptr(), vs[0] if layers else 0, vs[lead + 1], vs[lead], cu_seqlens.data_ptr(), total,
          max_seqlen, context.data_ptr(), ctx_sb, _ptr(cos), _ptr(sin), cs_sn, pool, b, HEAD_DIM)


def read_paged8(pools, block_table: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                first: torch.Tensor, lengths=None, total: int | None = None):
    """Slots of rows back in fp16: row b's slots [first[b], first[b] +
    cu_seqlens[b + 1] - cu_seqlens[b]), packed.

    ``cu_seqlens`` (B + 1,) int32, ``max_seqlen`` and ``lengths`` as in
    ``append_paged8``, ``first`` (B,) int64 read on the device.  ``total``: tokens of
    the result (default: the sum of ``lengths``, or the last of ``cu_seqlens``, which
    is then read from the device).  A row with a negative first, and slots past a
    row's pages, give zeros.  Returns k and v (T, KVH, 64), or (layers, T, KVH, 64)
    for ``PagedKv8Cache.all_pools``.
    """
    k = pools[0] if isinstance(pools, (tuple, list)) and len(pools) == 4 else None
    if not isinstance(k, torch.Tensor) or not k.is_cuda or k.dim() not in (4, 5):
        raise RuntimeError("pools must be (k, v, k_scale, v_scale) HIP device tensors; there is no CPU path")
    index, layers = k.get_device(), k.shape[0] if k.dim() == 5 else 0
    if total is None:
        total = sum(lengths) if lengths is not None else int(cu_seqlens[-1])
    b, first_sb = _packed(cu_seqlens, total, max_seqlen, first, "first", index, lengths)
    pool, _ = _pools8(pools, block_table, b, index, layers)
    shape = (2, layers or 1, total, pool.KVH, HEAD_DIM)
    out = torch.empty(shape, device=k.device, dtype=torch.float16)
    step = total * pool.KVH * HEAD_DIM
    at = out.data_ptr()
    _call("qf_read_paged8", index, at, step, HEAD_DIM, pool.KVH * HEAD_DIM, at + 2 * step * (layers or 1), step,
          HEAD_DIM, pool.KVH * HEAD_DIM, cu_seqlens.data_ptr(), total, max_seqlen, first.data_ptr(), first_sb,
          pool, b, HEAD_DIM)
    k, v = out.unbind(0)
    return (k, v) if layers else (k[0], v[0])


def copy_pages8(store: torch.Tensor, src, dst) -> None:
    """Page ``dst[i]`` becomes page ``src[i]`` in every layer of a
    ``PagedKv8Cache.store``, in one launch.

    ``src`` and ``dst`` are int32 device tensors (n,), read when the kernel runs, or
    sequences of ints, as in ``paged.copy_pages``."""
    if not isinstance(store, torch.Tensor) or not store.is_cuda:
        raise RuntimeError("store must be a HIP device tensor; there is no CPU path")
    if store.dtype is not torch.uint8 or store.dim() != 3 or not store.is_contiguous():
        raise ValueError("store must be a contiguous (layers, n_pages, bytes) uint8 tensor")
    layers, n_pages, size = store.shape
    index = store.get_device()
    if isinstance(src, torch.Tensor) and src.is_cuda:
        n = src.numel()
        for name, t in (("src", src), ("dst", dst)):
            if _int_rows(name, t, n, torch.int32, index) != 1 and n > 1:
                raise ValueError(f"{name} must be contiguous")
    else:
        if any(isinstance(t, torch.Tensor) and t.is_cuda for t in (src, dst)):
            raise TypeError("src and dst must both be device tensors or both sequences of ints")
        n = len(src)
        a, b = _page_list("src", src, n, 0, n_pages), _page_list("dst", dst, n, 0, n_pages)
        if len(set(b)) != n or set(a) & set(b):
            raise ValueError("no page may be written twice, or both written and read")
        src, dst = torch.tensor([a, b], dtype=torch.int32).to(store.device)
    _call("qf_copy_pages8", index, store.data_ptr(), layers, n_pages * size, size, size, src.data_ptr(),
          dst.data_ptr(), n, n_pages)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def _decode_args(grouped, pools, block_table, kv_last):
    _half("grouped", grouped, 4)
    b, kvh, _, _ = grouped.shape
    index = grouped.get_device()
    pool, cap = _pools8(pools, block_table, b, index)
    if pool.KVH != kvh:
        raise ValueError(f"pools hold {pool.KVH} kv heads, grouped {kvh}")
    return index, pool, cap, _int_rows("kv_last", kv_last, b, torch.int64, index)


def flash_decode_attention_paged8(grouped: torch.Tensor, pools, block_table: torch.Tensor,
                                  kv_last: torch.Tensor, scale: float | None = None,
                                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of a batch over pages held in 8 bits.

    grouped (B, KVH, G, 64) fp16, G at most 16; ``pools`` one layer's; block_table (B,
    pages_per_row) int32; ``kv_last`` (B,) int64 is each row's last slot, read on the
    device, and a row with a negative one (parked) gets zeros.  ``scale`` defaults to
    64 ** -0.5.  Returns (B, KVH, G, 64), written to ``out`` if given.  A row's result
    does not depend on the other rows.
    """
    index, pool, cap, last_sb = _decode_args(grouped, pools, block_table, kv_last)
    b, kvh, g, d = grouped.shape
    if out is None:
        out = (torch.empty_like(grouped) if grouped.is_contiguous()
               else torch.empty((b, kvh, g, d), device=grouped.device, dtype=torch.float16))
    else:
        _half("out", out, 4)
        if out.shape != grouped.shape or out.get_device() != index:
            raise ValueError(f"out must be {tuple(grouped.shape)} on {grouped.device}")
    need = _lib.load().qf_decode_attn_paged8_workspace(b, kvh, g, cap)
    ws = None if need == 0 else _workspace(need, "qf_decode_attn_paged8_workspace", grouped.device)
    _call("qf_decode_attn_paged8", index, grouped.data_ptr(), *grouped.stride()[:3], pool, kv_last.data_ptr(),
          last_sb, _ptr(ws), max(need, 0), out.data_ptr(), *out.stride()[:3], b, g, d,
          d ** -0.5 if scale is None else scale)
    return out


def flash_decode_split_paged8(grouped: torch.Tensor, pools, block_table: torch.Tensor, flash,
                              kv_last: torch.Tensor, scale: float | None = None):
    """The split launch alone: fills ``flash[0:3]`` = (acc, m, l) of
    ``ops.make_flash_scratch``, for ``ops.flash_decode_combine`` or
    ``step_ops.attn_merge_o_proj``."""
    index, pool, cap, last_sb = _decode_args(grouped, pools, block_table, kv_last)
    acc, m, l, _, _, splits, _, _ = _scratch_args(grouped, cap, None, flash, kv_last)
    b, _, g, d = grouped.shape
    _call("qf_decode_split_paged8", index, grouped.data_ptr(), *grouped.stride()[:3], pool, kv_last.data_ptr(),
          last_sb, acc.data_ptr(), m.data_ptr(), l.data_ptr(), splits, b, g, d,
          d ** -0.5 if scale is None else scale)
    return acc, m, l


def prefill_extend_paged8(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                          cu_seqlens: torch.Tensor, max_seqlen: int, context: torch.Tensor,
                          cos: torch.Tensor | None, sin: torch.Tensor | None, pools,
                          block_table: torch.Tensor, lengths=None, max_slots: int | None = None,
                          scale: float | None = None) -> torch.Tensor:
    """New tokens appended to rows that hold slots already, and attended.

    ``append_paged8`` of key and value, then token i of row b, packed query (T, QH,
    64), attends to slots [0, context[b] + i] as the pages hold them, its own and the
    call's other tokens among them.  ``cos``/``sin`` rotate query and key.
    ``max_slots`` bounds every row's context + tokens (default: the table's): the work
    is split by it, and slots past it are neither written nor read.  A parked row
    (negative context) gets zeros.  Returns (T, QH, 64).
    """
    _half("query", query, 3)
    _half("key", key, 3)
    _half("value", value, 3)
    total, qh, d = query.shape
    kvh = key.shape[1]
    if key.shape[0] != total or value.shape != key.shape or kvh < 1 or qh % kvh != 0:
        raise ValueError("packed extension shapes: query (T, QH, D), key/value (T, KVH, D)")
    index = query.get_device()
    if key.get_device() != index or value.get_device() != index:
        raise ValueError(f"query, key and value must be on one device ({query.device})")
    b, ctx_sb = _packed(cu_seqlens, total, max_seqlen, context, "context", index, lengths)
    pool, cap = _pools8(pools, block_table, b, index)
    if pool.KVH != kvh:
        raise ValueError(f"pools hold {pool.KVH} kv heads, key {kvh}")
    if max_slots is not None:
        if not max_seqlen <= max_slots <= cap:
            raise ValueError(f"max_slots must be in [{max_seqlen}, {cap}] (got {max_slots})")
        cap = int(max_slots)
    elif max_seqlen > cap:
        raise ValueError(f"max_seqlen exceeds the row capacity {cap}")
    cos, sin, cs_sn = _rope(cos, sin, total, index)
    out = torch.empty((total, qh, d), device=query.device, dtype=torch.float16)
    need = _lib.load().qf_prefill_extend_paged8_workspace(b, qh, kvh, total, max_seqlen, cap)
    ws = None if need == 0 else _workspace(need, "qf_prefill_extend_paged8_workspace", query.device)
    qs, ks, vs = query.stride(), key.stride(), value.stride()
    _call("qf_prefill_extend_paged8", index, query.data_ptr(), qs[1], qs[0], key.data_ptr(), ks[1], ks[0],
          value.data_ptr(), vs[1], vs[0], cu_seqlens.data_ptr(), total, max_seqlen, context.data_ptr(), ctx_sb,
          _ptr(cos), _ptr(sin), cs_sn, pool, cap, _ptr(ws), max(need, 0), out.data_ptr(), d, qh * d, b, qh, d,
          d ** -0.5 if scale is None else scale)
    return out
