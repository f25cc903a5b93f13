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

import functools
import struct

import torch

from . import _lib, paged
from .ops import HEAD_DIM, _require_cuda_fp16, _scratch_args
from .paged import MAX_PAGE, _check_page_size, _check_rows, _int_rows, _page_list

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

# The structs of the C ABI, all of 8-byte fields: packed here in one go, where
# handing that many arguments to ctypes would take longer than the launch.
POOL = struct.Struct("=18q")
_ROWS = struct.Struct("=36q")         # QfPool8 (18), then QfRows8's own
_DECODE = struct.Struct("=39qd")      # QfPool8, then QfDecode8's own
_EXTEND = struct.Struct("=46qd")      # QfRows8, then QfExtend8's own


def _explain_pools(pools, index: int, lead: int) -> None:
    """Raises for what ``_pools8`` refused."""
    if not isinstance(pools, (tuple, list)) or len(pools) != 4:
        raise TypeError("pools must be (k, v, k_scale, v_scale)")
    k, v, ks, vs = pools
    for name, t in zip(("k", "v", "k_scale", "v_scale"), pools):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
            raise RuntimeError(f"{name} must be a tensor on cuda:{index}; there is no CPU path")
    if k.dtype not in _KINDS or v.dtype is not k.dtype or ks.dtype is not torch.float32 \
            or vs.dtype is not torch.float32:
        raise TypeError("k and v must both be int8 or float8_e4m3fn, k_scale and v_scale float32 "
                        f"(got {k.dtype}, {v.dtype}, {ks.dtype}, {vs.dtype})")
    shape = tuple(k.shape)
    if len(shape) != 4 + lead or 0 in shape or shape[-1] != HEAD_DIM:
        raise ValueError(f"k must be {'(layers, ' if lead else '('}n_pages, KVH, P, 64) (got {shape})")
    page, outer = shape[-2], shape[:lead + 2]
    _check_page_size(page)
    if v.shape != (*outer, page // 64, HEAD_DIM, 64) or ks.shape != (*outer, page // BLOCK) or vs.shape != ks.shape:
        raise ValueError(f"pools of {outer} pages and heads of {page} slots need v (.., P / 64, 64, 64) and "
                         f"scales (.., P / {BLOCK})")
    raise ValueError("k and v must have the same page and head strides, and so must the scales; "
                     "what a page and head holds must be contiguous")


def _pools8(pools, block_table, batch: int, index: int, lead: int = 0):
    """``QfPool8``'s fields for a layer's pools -- with ``lead`` 1 for all layers', as
    ``PagedKv8Cache.all_pools`` -- and the rows' table on GPU ``index``; the pools' kv
    heads and the slots of a row.  Reads as few tensor properties as it can and
    explains itself only when it refuses."""
    try:
        k, v, ks, vs = pools
        shape, strides, scale_strides = k.shape, k.stride(), ks.stride()
        if lead:
            layers, n_pages, kvh, page, d = shape
            head, outer, scale_outer = (layers, n_pages, kvh), strides[:3], scale_strides[:3]
        else:
            n_pages, kvh, page, d = shape
            layers, head, outer, scale_outer = 1, (n_pages, kvh), strides[:2], scale_strides[:2]
        dtype, scale_shape = k.dtype, (*head, page // BLOCK)
        kind = _KINDS[dtype]
        ok = (d == HEAD_DIM and n_pages > 0 and kvh > 0 and layers > 0
              and 64 <= page <= MAX_PAGE and not page & (page - 1)
              and v.shape == (*head, page // 64, HEAD_DIM, 64) and ks.shape == scale_shape
              and vs.shape == scale_shape and v.dtype is dtype
              and ks.dtype is torch.float32 and vs.dtype is torch.float32
              and strides == (*outer, 64, 1) and v.stride() == (*outer, 4096, 64, 1)
              and scale_strides == (*scale_outer, 1) and vs.stride() == scale_strides
              and k.get_device() == v.get_device() == ks.get_device() == vs.get_device() == index >= 0)
    except (AttributeError, KeyError, TypeError, ValueError):
        ok = False
    if not ok:
        _explain_pools(pools, index, lead)
    try:
        (rows, ppr), (table_sb, unit) = block_table.shape, block_table.stride()
        if block_table.dtype is not torch.int32 or block_table.get_device() != index:
            raise TypeError(f"block_table must be an int32 tensor on cuda:{index}")
    except AttributeError:
        raise TypeError(f"block_table must be an int32 tensor on cuda:{index}") from None
    except ValueError:
        rows = unit = -1
    if rows != batch or unit != 1:
        raise ValueError(f"block_table must be (B={batch}, pages_per_row) with unit inner stride")
    if not lead:
        outer, scale_outer = (0, *outer), (0, *scale_outer)
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *outer, *scale_outer,
            block_table.data_ptr(), table_sb, ppr, n_pages, page, layers, kvh, kind), kvh, ppr * page


def _call8(name: str, index: int, *args) -> None:
    """Entry point ``name`` on GPU ``index`` and its current stream."""
    fn = getattr(_lib.load(), name)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name: str, *sizes) -> int:
    need = getattr(_lib.load(), name)(*sizes)
    if need < 0:
        _lib.check(need, name)
    return need


def _scratch(need: int, device):
    return torch.empty(need, device=device, dtype=torch.uint8) if need else None


def _half8(name: str, t, ndim: int):
    """Shape and strides of an fp16 device tensor of ``ndim`` dimensions with 64 contiguous
    values in the last, or raises."""
    try:
        shape, strides = t.shape, t.stride()
        if t.dtype is torch.float16 and len(shape) == ndim and shape[-1] == HEAD_DIM and strides[-1] == 1 \
                and t.get_device() >= 0:
            return shape, strides
    except (AttributeError, IndexError):
        pass
    _require_cuda_fp16(name, t, ndim)
    raise RuntimeError(f"{name} must be a HIP device tensor")


def _ints8(name: str, t, n: int, dtype, index: int) -> int:
    """Stride of an ``(n,)`` tensor of ``dtype`` on GPU ``index``, or raises."""
    try:
        if t.dtype is dtype and t.shape == (n,) and t.get_device() == index:
            return t.stride()[0]
    except AttributeError:
        pass
    return _int_rows(name, t, n, dtype, index)


def _packed(cu_seqlens, total: int, max_seqlen: int, first, name: str, index: int, lengths):
    """Rows of packed tokens and each one's first slot: their number and first's stride."""
    try:
        (b,) = cu_seqlens.shape
        b -= 1
    except (AttributeError, ValueError):
        b = 0
    if b < 1 or not 1 <= max_seqlen <= total:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    if _ints8("cu_seqlens", cu_seqlens, b + 1, torch.int32, index) != 1:
        raise ValueError("cu_seqlens must be contiguous")
    stride = _ints8(name, first, b, torch.int64, index)
    _check_rows(cu_seqlens, total, max_seqlen, lengths)
    return b, stride


def _rope(cos, sin, total: int, index: int):
    """(cos, sin, token stride) of per-token tables (T, 64), or Nones."""
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is None:
        return None, None, 0
    for n, t in (("cos", cos), ("sin", sin)):
        _half8(n, t, 2)
        if t.shape[0] != total or t.get_device() != index:
            raise ValueError(f"{n} must be (T={total}, 64) on cuda:{index}")
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin, cos.stride(0)


def _address(t) -> int:
    return 0 if t is None else t.data_ptr()


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
    have no tokens; of one that the device's offsets make longer than ``max_seqlen``
    the first ``max_seqlen`` are taken); ``context`` (B,) int64 is read on the device, and a row with a
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
    lead = 1 if isinstance(key, torch.Tensor) and key.dim() == 4 else 0
    shape, ks = _half8("key", key, 3 + lead)
    other, vs = _half8("value", value, 3 + lead)
    index, total, kvh = key.get_device(), shape[lead], shape[lead + 1]
    if other != shape or value.get_device() != index:
        raise ValueError(f"key and value must be alike (got {tuple(shape)}, {tuple(other)})")
    b, ctx_sb = _packed(cu_seqlens, total, max_seqlen, context, "context", index, lengths)
    pool, heads, cap = _pools8(pools, block_table, b, index, lead)
    if heads != kvh or (lead and pool[15] != shape[0]):
        raise ValueError(f"pools of {pool[15]} layers and {heads} kv heads do not match key {tuple(shape)}")
    if max_seqlen > cap:
        raise ValueError(f"max_seqlen exceeds the row capacity {cap}")
    cos, sin, cs_sn = _rope(cos, sin, total, index)
    _call8("qf_append_paged8", index, _ROWS.pack(
        *pool, key.data_ptr(), ks[0] if lead else 0, ks[lead + 1], ks[lead], value.data_ptr(),
        vs[0] if lead else 0, vs[lead + 1], vs[lead], cu_seqlens.data_ptr(), total, max_seqlen,
        context.data_ptr(), ctx_sb, _address(cos), _address(sin), cs_sn, b, HEAD_DIM))


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
    index, lead = k.get_device(), k.dim() - 4
    if total is None:
        total = sum(lengths) if lengths is not None else int(cu_seqlens[-1])
    b, first_sb = _packed(cu_seqlens, total, max_seqlen, first, "first", index, lengths)
    pool, kvh, _ = _pools8(pools, block_table, b, index, lead)
    layers, row = pool[15], kvh * HEAD_DIM
    out = torch.empty((2, layers, total, kvh, HEAD_DIM) if lead else (2, total, kvh, HEAD_DIM),
                      device=k.device, dtype=torch.float16)
    at, step = out.data_ptr(), total * row
    _call8("qf_read_paged8", index, _ROWS.pack(
        *pool, at, step, HEAD_DIM, row, at + 2 * step * layers, step, HEAD_DIM, row, cu_seqlens.data_ptr(), total,
        max_seqlen, first.data_ptr(), first_sb, 0, 0, 0, b, HEAD_DIM))
    return out.unbind(0)


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
    _call8("qf_copy_pages8", index, store.data_ptr(), layers, n_pages * size, size, size, src.data_ptr(),
           dst.data_ptr(), n, n_pages)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def _decode_args(grouped, pools, block_table, kv_last, key, value):
    """``QfDecode8``'s fields up to kv_last's, the call's GPU, shape and capacity, and
    the fields of the new tokens."""
    shape, strides = _half8("grouped", grouped, 4)
    index = grouped.get_device()
    pool, kvh, cap = _pools8(pools, block_table, shape[0], index)
    if kvh != shape[1]:
        raise ValueError(f"pools hold {kvh} kv heads, grouped {shape[1]}")
    last_sb = _ints8("kv_last", kv_last, shape[0], torch.int64, index)
    new = (0, 0, 0, 0, 0, 0)
    if (key is None) != (value is None):
        raise ValueError("key and value go together")
    if key is not None:
        k_shape, k_strides = _half8("key", key, 3)
        v_shape, v_strides = _half8("value", value, 3)
        if k_shape != (shape[0], kvh, HEAD_DIM) or v_shape != k_shape or not (
                key.get_device() == value.get_device() == index):
            raise ValueError(f"key and value must be {(shape[0], kvh, HEAD_DIM)} on cuda:{index}")
        new = (key.data_ptr(), k_strides[0], k_strides[1], value.data_ptr(), v_strides[0], v_strides[1])
    return (*pool, grouped.data_ptr(), strides[0], strides[1], strides[2], kv_last.data_ptr(),
            last_sb), index, shape, cap, new


def flash_decode_attention_paged8(grouped: torch.Tensor, pools, block_table: torch.Tensor,
                                  kv_last: torch.Tensor, scale: float | None = None,
                                  out: torch.Tensor | None = None, key: torch.Tensor | None = None,
                                  value: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of a batch over pages held in 8 bits.

    grouped (B, KVH, G, 64) fp16, G at most 16; ``pools`` one layer's; block_table (B,
    pages_per_row) int32; ``kv_last`` (B,) int64 is each row's last slot, read on the
    device, and a row with a negative one (parked) gets zeros.  ``scale`` defaults to
    64 ** -0.5.  Returns (B, KVH, G, 64), written to ``out`` if given.  A row's result
    does not depend on the other rows.

    With ``key`` and ``value`` (B, KVH, 64) each row's new token is first appended at slot
    kv_last, as ``append_paged8`` does, in the same launch: a decoding step's.
    """
    head, index, shape, cap, new = _decode_args(grouped, pools, block_table, kv_last, key, value)
    b, kvh, g, d = shape
    device = grouped.device
    if out is None:
        out = torch.empty(shape, device=device, dtype=torch.float16)
        strides = (kvh * g * d, g * d, d)
    else:
        o_shape, strides = _half8("out", out, 4)
        if o_shape != shape or out.get_device() != index:
            raise ValueError(f"out must be {tuple(shape)} on {device}")
    need = _workspace_bytes("qf_decode_attn_paged8_workspace", b, kvh, g, cap)
    ws = _scratch(need, device)
    _call8("qf_decode_attn_paged8", index, _DECODE.pack(
        *head, out.data_ptr(), strides[0], strides[1], strides[2], _address(ws), need, b, g, d, *new,
        d ** -0.5 if scale is None else scale))
    return out


def flash_decode_split_paged8(grouped: torch.Tensor, pools, block_table: torch.Tensor, flash,
                              kv_last: torch.Tensor, scale: float | None = None,
                              key: torch.Tensor | None = None, value: torch.Tensor | None = None):
    """The split launch alone: fills ``flash[0:3]`` = (acc, m, l) of
    ``ops.make_flash_scratch``, for ``ops.flash_decode_combine`` or
    ``step_ops.attn_merge_o_proj``; ``key`` and ``value`` as in
    ``flash_decode_attention_paged8``."""
    head, index, (b, _, g, d), cap, new = _decode_args(grouped, pools, block_table, kv_last, key, value)
    acc, m, l, _, _, splits, _, _ = _scratch_args(grouped, cap, None, flash, kv_last)
    _call8("qf_decode_split_paged8", index, _DECODE.pack(
        *head, 0, 0, 0, 0, 0, 0, b, g, d, *new, d ** -0.5 if scale is None else scale),
        acc.data_ptr(), m.data_ptr(), l.data_ptr(), splits)
    return acc, m, l


def prefill_extend_paged8(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                          cu_seqlens: torch.Tensor, max_seqlen: int, context: torch.Tensor,
                          cos: torch.Tensor | None, sin: torch.Tensor | None, pools,
                          block_table: torch.Tensor, lengths=None, max_slots: int | None = None,
                          scale: float | None = None) -> torch.Tensor:
    """New tokens appended to rows that hold slots already, and attended.

    ``append_paged8`` of key and value, then token i of row b, packed query (T, QH,
    64), attends to slots [0, context[b] + i] as the pages hold them, its own and the
    call's other tokens among them.  QH is at most 16 times key's heads.
    ``cos``/``sin`` rotate query and key.
    ``max_slots`` bounds every row's context + tokens (default: the table's): the work
    is split by it, and slots past it are neither written nor read.  A parked row
    (negative context) gets zeros.  Returns (T, QH, 64).
    """
    (total, qh, d), qs = _half8("query", query, 3)
    shape, ks = _half8("key", key, 3)
    v_shape, vs = _half8("value", value, 3)
    kvh = shape[1]
    if shape[0] != total or v_shape != shape or kvh < 1 or qh % kvh != 0:
        raise ValueError("packed extension shapes: query (T, QH, D), key/value (T, KVH, D)")
    index = query.get_device()
    if key.get_device() != index or value.get_device() != index:
        raise ValueError(f"query, key and value must be on one device ({query.device})")
    b, ctx_sb = _packed(cu_seqlens, total, max_seqlen, context, "context", index, lengths)
    pool, heads, cap = _pools8(pools, block_table, b, index)
    if heads != kvh:
        raise ValueError(f"pools hold {heads} kv heads, key {kvh}")
    if max_slots is not None:
        if not max_seqlen <= max_slots <= cap:
            raise ValueError(f"max_slots must be in [{max_seqlen}, {cap}] (got {max_slots})")
        cap = int(max_slots)
    elif max_seqlen > cap:
        raise ValueError(f"max_seqlen exceeds the row capacity {cap}")
    cos, sin, cs_sn = _rope(cos, sin, total, index)
    device = query.device
    out = torch.empty((total, qh, d), device=device, dtype=torch.float16)
    need = _workspace_bytes("qf_prefill_extend_paged8_workspace", b, qh, kvh, total, max_seqlen, cap)
    ws = _scratch(need, device)
    _call8("qf_prefill_extend_paged8", index, _EXTEND.pack(
        *pool, key.data_ptr(), 0, ks[1], ks[0], value.data_ptr(), 0, vs[1], vs[0], cu_seqlens.data_ptr(), total,
        max_seqlen, context.data_ptr(), ctx_sb, _address(cos), _address(sin), cs_sn, b, d, query.data_ptr(), qs[1],
        qs[0], out.data_ptr(), d, qh * d, cap, _address(ws), need, qh, d ** -0.5 if scale is None else scale))
    return out
