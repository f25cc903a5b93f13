"""Paged KV cache: page pools, block tables and the paged attention-path ops.

The reference engine keeps one dense ``(B, KVH, cap, 64)`` cache per layer
and right-pads ragged batches (SE:1162-1204, SE:1263-1319); block-level KV
management is on its roadmap ("PagedAttention & Continuous Batching",
README.md:144).  Here the caches of all layers are page pools
``(n_pages, KVH, page_size, 64)`` fp16 and one int32 block table per batch
maps a row's logical pages to physical pages, so rows have no padding holes
and can be admitted and retired independently.  The ops call the C ABI in
``include/qf_paged.h``; like ``ops``, nothing computes on the host.

* ``PagedKvCache`` -- pools for every layer, the device block table and a
  host free list of pages; rows forked from one another share whole pages.
* ``copy_pages`` -- pages of every layer copied to other pages in one launch.
* ``flash_decode_attention_paged`` / ``flash_decode_split_paged`` -- split-K
  decode (SE:834-874 semantics) through the block table.
* ``flash_decode_attention_prefix_paged`` -- decode of a batch whose rows share
  prefixes, which are read once.
* ``rope_append_paged`` -- one-token RoPE + append at a per-row slot.
* ``prefill_varlen_paged`` -- packed ragged prefill appending into pages.
* ``prefill_extend_paged`` -- packed new tokens of rows that hold slots already.
* ``rms_qkv_rope_append_paged`` -- the fused decode-step QKV kernel appending
  into pages.
"""

from __future__ import annotations

import ctypes as C
import operator

import torch

from . import _lib
from .ops import HEAD_DIM, _ptr, _require_cuda_fp16, _scratch_args, _stream, check_cu_seqlens
from .step_ops import PACK_ROPE, _batch, _check, _rows, _weight, rope_args

MIN_PAGE, MAX_PAGE = 64, 4096


def _check_page_size(page_size: int) -> None:
    if not MIN_PAGE <= page_size <= MAX_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two in [{MIN_PAGE}, {MAX_PAGE}] (got {page_size})")


class PagedKvCache:
    """Page pools of ``layers`` layers plus the block table of up to ``max_rows`` rows.

    ``pools[i] = (k_pool, v_pool)``, each ``(n_pages, kv_heads, page_size, 64)``
    fp16, zero-initialised views of the one contiguous allocation ``store``
    (layers, 2, n_pages, kv_heads, page_size, 64).  ``table`` is ``(max_rows, pages_per_row)``
    int32 on the device; unmapped entries hold -1.  Pages are handed out from a
    host free list (lowest id first); ``map_row`` / ``release_row`` update the
    device table with one small copy each, so they belong between graph
    replays, not inside them.

    ``fork_rows`` maps the whole pages of a row into other rows too: such a page
    is shared, and goes back to the free list with the last row that holds it.
    Nothing may be written to a shared page: a row that will write to slots it
    shares takes the pages for itself first (``own_slots``).  The slots after a
    fork's are its own.  Like ``map_row`` these belong between graph replays and
    on the stream that the cache's kernels run on.
    """

    def __init__(self, layers: int, kv_heads: int, n_pages: int, page_size: int, max_rows: int,
                 pages_per_row: int, device, dtype=torch.float16):
        _check_page_size(page_size)
        if n_pages < 1 or max_rows < 1 or pages_per_row < 1:
            raise ValueError("need n_pages, max_rows and pages_per_row >= 1")
        self.page_size = page_size
        self.n_pages = n_pages
        self.kv_heads = kv_heads
        self.pages_per_row = pages_per_row
        self.device = torch.device(device)
        self.store = torch.zeros((layers, 2, n_pages, kv_heads, page_size, HEAD_DIM),
                                 device=self.device, dtype=dtype)
        self.pools = [(layer[0], layer[1]) for layer in self.store]
        self.table = torch.full((max_rows, pages_per_row), -1, device=self.device, dtype=torch.int32)
        self._free = list(range(n_pages))
        self._rows: dict[int, list[int]] = {}
        self._holders = [0] * n_pages          # rows that hold each page

    @property
    def capacity(self) -> int:
        """Logical slots per row."""
        return self.pages_per_row * self.page_size

    def free_pages(self) -> int:
        return len(self._free)

    def row_pages(self, row: int) -> list[int]:
        return list(self._rows.get(row, []))

    def map_row(self, row: int, n_slots: int) -> list[int]:
        """Make slots ``[0, n_slots)`` of ``row`` backed by pages (growing its
        mapping as needed); returns the row's page list."""
        need = -(-n_slots // self.page_size)
        if need > self.pages_per_row:
            raise ValueError(f"{n_slots} slots exceed the row capacity {self.capacity}")
        pages = self._rows.setdefault(row, [])
        if need - len(pages) > len(self._free):
            raise RuntimeError(f"page pool exhausted: need {need - len(pages)}, {len(self._free)} free")
        first = len(pages)
        while len(pages) < need:
            pages.append(self._take())
        if len(pages) > first:
            ids = torch.tensor(pages[first:], dtype=torch.int32)
            self.table[row, first:len(pages)].copy_(ids)
        return list(pages)

    def _take(self) -> int:
        page = self._free.pop(0)
        self._holders[page] = 1
        return page

    def release_row(self, row: int) -> None:
        """Unmap the row and return the pages that no other row holds to the
        free list."""
        pages = self._rows.pop(row, [])
        for page in pages:
            self._holders[page] -= 1
            if self._holders[page] == 0:
                self._free.append(page)
        self._free.sort()
        self.table[row].fill_(-1)

    def shared_pages(self, row: int) -> int:
        """Pages of ``row`` that another row holds too."""
        return sum(self._holders[p] > 1 for p in self._rows.get(row, []))

    def fork_rows(self, src: int, rows, n_slots: int) -> None:
        """Makes slots ``[0, n_slots)`` of row ``src`` those of every row of
        ``rows`` (unmapped before): whole pages are shared, a partly filled last
        page is copied into a page of the row's own, for all rows and layers in
        one launch.  ``map_row`` then grows the rows as usual."""
        rows = [operator.index(r) for r in rows]
        pages = self._rows.get(src, [])
        if not 0 <= n_slots <= len(pages) * self.page_size:
            raise ValueError(f"row {src} has {len(pages) * self.page_size} slots mapped, not {n_slots}")
        if len(set(rows)) != len(rows) or any(
                not 0 <= r < self.table.shape[0] or self._rows.get(r) for r in rows):
            raise ValueError("rows to fork into must be distinct rows of the table with nothing mapped")
        whole, rest = divmod(n_slots, self.page_size)
        if rest and len(rows) > len(self._free):
            raise RuntimeError(f"page pool exhausted: need {len(rows)}, {len(self._free)} free")
        own = self._free[:len(rows)] if rest else []
        if own:
            copy_pages(self.store, [pages[whole]] * len(rows), own, slots=[rest] * len(rows))
        for i, row in enumerate(rows):
            if rest:
                self._take()
            for page in pages[:whole]:
                self._holders[page] += 1
            self._rows[row] = pages[:whole] + own[i:i + 1]
        self._upload(rows)

    def fork_row(self, src: int, row: int, n_slots: int) -> None:
        """``fork_rows`` into one row."""
        self.fork_rows(src, [row], n_slots)

    def own_slots(self, row: int, first: int, n_slots: int) -> int:
        """Gives ``row`` pages of its own for slots ``[first, first + n_slots)``,
        copied from the shared ones it held there, so that it may write to them;
        returns how many pages were copied."""
        pages = self._rows.get(row, [])
        if first < 0 or n_slots < 0 or first + n_slots > len(pages) * self.page_size:
            raise ValueError(f"slots [{first}, {first + n_slots}) are not all mapped in row {row}")
        if n_slots == 0:
            return 0
        at = [j for j in range(first // self.page_size, (first + n_slots - 1) // self.page_size + 1)
              if self._holders[pages[j]] > 1]
        if len(at) > len(self._free):
            raise RuntimeError(f"page pool exhausted: need {len(at)}, {len(self._free)} free")
        if at:
            copy_pages(self.store, [pages[j] for j in at], self._free[:len(at)])
            for j in at:
                self._holders[pages[j]] -= 1
                pages[j] = self._take()
            self._upload([row])
        return len(at)

    def compact(self) -> int:
        """Moves the pages in use to the lowest ids, so that the free ones are
        the pool's end; returns how many moved.  Tables follow, shared pages
        stay shared."""
        used = [p for p, n in enumerate(self._holders) if n]
        src = [p for p in used if p >= len(used)]
        dst = [p for p in self._free if p < len(used)]
        if not src:
            return 0
        copy_pages(self.store, src, dst)
        to = dict(zip(src, dst))
        for pages in self._rows.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        self._free = list(range(len(used), self.n_pages))
        self._upload(self._rows)
        return len(src)

    def _upload(self, rows) -> None:
        """The device table's entries of ``rows``, from the host lists, in one copy."""
        rows = list(rows)
        if not rows:
            return
        host = torch.full((len(rows), self.pages_per_row), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            host[i, :len(self._rows[r])] = torch.tensor(self._rows[r], dtype=torch.int32)
        self.table.index_copy_(0, torch.tensor(rows, device=self.device), host.to(self.device))

    def gather(self, layer: int, row: int, length: int):
        """Slots ``[0, length)`` of ``row`` as dense ``(KVH, length, 64)`` K and V
        (device indexing; for inspection and tests)."""
        k_pool, v_pool = self.pools[layer]
        pages = torch.tensor(self._rows[row], device=self.device, dtype=torch.long)
        slot = torch.arange(length, device=self.device)
        page = pages[slot // self.page_size]
        off = slot % self.page_size
        return k_pool[page, :, off].transpose(0, 1), v_pool[page, :, off].transpose(0, 1)


# --------------------------------------------------------------------------
# argument helpers
# --------------------------------------------------------------------------

def _pool_args(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, batch: int):
    """Validate the pools and the (B, pages_per_row) table; returns the ABI pieces."""
    _require_cuda_fp16("k_pool", k_pool, 4)
    _require_cuda_fp16("v_pool", v_pool, 4)
    if v_pool.shape != k_pool.shape:
        raise ValueError("k_pool and v_pool must have the same shape")
    n_pages, _, page_size, _ = k_pool.shape
    _check_page_size(page_size)
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.device != k_pool.device:
        raise RuntimeError("block_table must be on the pools' device")
    if block_table.dim() != 2 or block_table.shape[0] != batch or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be (B={batch}, pages_per_row) with unit inner stride")
    ppr = block_table.shape[1]
    return ((k_pool.data_ptr(), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2),
             v_pool.data_ptr(), v_pool.stride(0), v_pool.stride(1), v_pool.stride(2),
             block_table.data_ptr(), block_table.stride(0), ppr, n_pages, page_size),
            ppr * page_size)


# The calls below serve single tokens, where a microsecond on the host counts:
# checks read as few tensor properties as they can and explain themselves only
# when they fail.

def _half(name: str, t: torch.Tensor, ndim: int) -> None:
    """``_require_cuda_fp16`` for a tensor that is expected to pass."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.float16 and t.is_cuda and t.dim() == ndim
            and t.shape[-1] == HEAD_DIM and t.stride(-1) == 1):
        _require_cuda_fp16(name, t, ndim)


def _int_rows(name: str, t: torch.Tensor, n: int, dtype, index: int) -> int:
    """Element stride of an ``(n,)`` tensor of ``dtype`` on GPU ``index``, or raises."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index:
        raise TypeError(f"{name} must be an {str(dtype)[6:]} tensor on cuda:{index}")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be ({n},) (got {tuple(t.shape)})")
    return t.stride(0)


def _pools(k_pool, v_pool, block_table, batch: int, kv_heads: int, index: int):
    """``_pool_args`` for ``kv_heads`` heads on GPU ``index``."""
    _half("k_pool", k_pool, 4)
    _half("v_pool", v_pool, 4)
    shape, ks, vs = k_pool.shape, k_pool.stride(), v_pool.stride()
    n_pages, kvh, page, _ = shape
    if v_pool.shape != shape or kvh != kv_heads or k_pool.get_device() != index \
            or v_pool.get_device() != index:
        raise ValueError(f"k_pool and v_pool must be alike and hold {kv_heads} kv heads on cuda:{index}")
    _check_page_size(page)
    if (not isinstance(block_table, torch.Tensor) or block_table.dtype is not torch.int32
            or block_table.get_device() != index):
        raise TypeError(f"block_table must be an int32 tensor on cuda:{index}")
    if block_table.dim() != 2 or block_table.shape[0] != batch or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be (B={batch}, pages_per_row) with unit inner stride")
    ppr = block_table.shape[1]
    return ((k_pool.data_ptr(), *ks[:3], v_pool.data_ptr(), *vs[:3], block_table.data_ptr(),
             block_table.stride(0), ppr, n_pages, page), ppr * page)


def _call(name: str, index: int, *args) -> None:
    """Entry point ``name`` on GPU ``index`` and its current stream."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, name)


def _check_rows(cu_seqlens, total: int, max_seqlen: int, lengths) -> None:
    """``check_cu_seqlens``; host lengths that are right are not walked through."""
    if (lengths is None or len(lengths) != cu_seqlens.shape[0] - 1 or sum(lengths) != total
            or min(lengths) < 0 or max(lengths) > max_seqlen):
        check_cu_seqlens(cu_seqlens, total, max_seqlen, lengths)


def _slot_args(slots: torch.Tensor, batch: int, device):
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int64 or slots.device != device:
        raise TypeError("slots must be an int64 device tensor")
    if slots.dim() != 1 or slots.numel() != batch:
        raise ValueError(f"slots must hold one slot per row ({batch})")
    return slots.data_ptr(), slots.stride(0)


# --------------------------------------------------------------------------
# page copies
# --------------------------------------------------------------------------

def _page_list(name: str, pages, n: int, low: int, high: int) -> list:
    pages = [operator.index(p) for p in pages]
    if len(pages) != n or any(not low <= p < high for p in pages):
        raise ValueError(f"{name} must be {n} whole numbers in [{low}, {high})")
    return pages


def copy_pages(pools, src, dst, slots=None) -> None:
    """Page ``dst[i]`` becomes page ``src[i]`` -- its first ``slots[i]`` slots, all
    of them without ``slots`` -- in every pool, in one launch.

    ``pools``: a contiguous tensor (..., n_pages, KVH, P, 64) fp16 such as
    ``PagedKvCache.store``, or a list of pools (n_pages, KVH, P, 64) of one
    layout.  ``src``, ``dst`` and ``slots`` are all int32 device tensors (n,),
    read when the kernel runs, or all sequences of ints.  Sequences are checked;
    with device tensors a pair with a page outside the pool copies nothing, a
    slot count is clamped to the page, and the caller sees to it that no page is
    written twice or both written and read.
    """
    if isinstance(pools, torch.Tensor):
        if pools.dim() < 4 or not pools.is_contiguous():
            raise ValueError("pools must be a contiguous (..., n_pages, KVH, P, 64) tensor, or a list")
        _half("pools", pools, pools.dim())
        first, shape, stride = pools, pools.shape[-4:], pools.stride()[-4:]
        step = shape[0] * stride[0]
        per = pools.numel() // step if step else 0
        bases = (pools.data_ptr(),)
    else:
        pools = list(pools)
        if not pools:
            raise ValueError("copy_pages needs at least one pool")
        first, per, step = pools[0], 1, 0
        for t in pools:
            _require_cuda_fp16("pool", t, 4)
            if t.shape != first.shape or t.stride() != first.stride() or t.device != first.device:
                raise ValueError("pools must have one shape, layout and device")
        shape, stride, bases = first.shape, first.stride(), [t.data_ptr() for t in pools]
    n_pages, kvh, page, _ = shape
    _check_page_size(page)
    if per < 1 or n_pages < 1 or kvh < 1:
        raise ValueError("copy_pages needs at least one pool, page and head")
    index = first.get_device()
    if isinstance(src, torch.Tensor) and src.is_cuda:
        n = src.numel()
        for name, t in (("src", src), ("dst", dst), ("slots", slots)):
            if t is not None or name != "slots":
                if _int_rows(name, t, n, torch.int32, index) != 1 and n > 1:
                    raise ValueError(f"{name} must be contiguous")
    else:
        if any(isinstance(t, torch.Tensor) and t.is_cuda for t in (src, dst, slots)):
            raise TypeError("src, dst and slots must all be device tensors or all sequences of ints")
        n = len(src)
        a, b = _page_list("src", src, n, 0, n_pages), _page_list("dst", dst, n, 0, n_pages)
        if len(set(b)) != n or set(a) & set(b):
            raise ValueError("no page may be written twice, or both written and read")
        rows = [a, b] + ([_page_list("slots", slots, n, 0, page + 1)] if slots is not None else [])
        up = torch.tensor(rows, dtype=torch.int32).to(first.device)
        src, dst, slots = up[0], up[1], up[2] if slots is not None else None
    _call("qf_copy_pages", index, (C.c_void_p * len(bases))(*bases), len(bases), per, step, stride[0],
          stride[1], stride[2], src.data_ptr(), dst.data_ptr(), _ptr(slots), n, n_pages, kvh, page, HEAD_DIM)


# --------------------------------------------------------------------------
# decode
# --------------------------------------------------------------------------

def _paged_decode_args(grouped, k_pool, v_pool, block_table, attn_bias, flash, kv_last):
    b = grouped.shape[0]
    pool, cap = _pool_args(k_pool, v_pool, block_table, b)
    kvh = grouped.shape[1]
    if k_pool.shape[1] != kvh:
        raise ValueError(f"pools hold {k_pool.shape[1]} kv heads, grouped {kvh}")
    acc, m, l, out, ticket, splits, _, kv_last_sb = _scratch_args(
        grouped, cap, attn_bias, flash, kv_last)
    head = (grouped.data_ptr(), grouped.stride(0), grouped.stride(1), grouped.stride(2))
    bias = (_ptr(attn_bias), 0 if attn_bias is None else attn_bias.stride(0),
            _ptr(kv_last), kv_last_sb)
    return head, pool, bias, acc, m, l, out, ticket, splits


def flash_decode_attention_paged(grouped: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                                 block_table: torch.Tensor, attn_bias: torch.Tensor | None, flash,
                                 kv_last: torch.Tensor | None = None, scale: float | None = None,
                                 share_rows: bool = True) -> torch.Tensor:
    """``flash_decode_attention`` over paged caches (SE:834-874 semantics).

    grouped (B, KVH, G, 64); pools (n_pages, KVH, P, 64); block_table
    (B, pages_per_row) int32; attn_bias (B, pages_per_row * P) or None;
    ``flash`` as in ``ops.make_flash_scratch``; kv_last (1,) or (B,) int64
    bounds each row's slots; ``share_rows`` as in
    ``ops.flash_decode_attention``.  Writes and returns ``flash[3]``.
    """
    head, pool, bias, acc, m, l, out, ticket, splits = _paged_decode_args(
        grouped, k_pool, v_pool, block_table, attn_bias, flash, kv_last)
    b, kvh, g, d = grouped.shape
    scale = d ** -0.5 if scale is None else scale
    name = "qf_decode_attn_paged_shared" if share_rows else "qf_decode_attn_paged"
    with torch.cuda.device(grouped.device):
        rc = getattr(_lib.load(), name)(
            *head, *pool, *bias, acc.data_ptr(), m.data_ptr(), l.data_ptr(), splits, _ptr(ticket),
            out.data_ptr(), out.stride(0), out.stride(1), out.stride(2),
            b, kvh, g, d, float(scale), _stream(grouped.device))
    _lib.check(rc, name)
    return out


def flash_decode_split_paged(grouped, k_pool, v_pool, block_table, attn_bias, flash, kv_last=None,
                             scale=None):
    """The split launch alone over paged caches: fills ``flash[0:3]`` = (acc, m, l)."""
    head, pool, bias, acc, m, l, _, _, splits = _paged_decode_args(
        grouped, k_pool, v_pool, block_table, attn_bias, flash, kv_last)
    b, kvh, g, d = grouped.shape
    scale = d ** -0.5 if scale is None else scale
    with torch.cuda.device(grouped.device):
        rc = _lib.load().qf_decode_split_paged(
            *head, *pool, *bias, acc.data_ptr(), m.data_ptr(), l.data_ptr(), splits,
            b, kvh, g, d, float(scale), _stream(grouped.device))
    _lib.check(rc, "qf_decode_split_paged")
    return acc, m, l


def _workspace(need: int, name: str, device) -> torch.Tensor:
    if need < 0:
        _lib.check(need, name)
    return torch.empty(max(need, 16), device=device, dtype=torch.uint8)


def flash_decode_attention_prefix_paged(grouped: torch.Tensor, k_pool: torch.Tensor,
                                        v_pool: torch.Tensor, block_table: torch.Tensor,
                                        prefix_rows: torch.Tensor, prefix_len: torch.Tensor,
                                        kv_last: torch.Tensor, scale: float | None = None,
                                        out: torch.Tensor | None = None,
                                        prefix_table: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of a batch whose rows share prefixes, each read once.

    grouped (B, KVH, G, 64), pools and block_table as in
    ``flash_decode_attention_paged``; ``prefix_rows`` (N + 1,) int32: rows
    [prefix_rows[g], prefix_rows[g + 1]) are group g, whose slots
    [0, prefix_len[g]) hold the same K and V in every row (forked rows'); they
    are read from the pages of the group's first row, or of row g of
    ``prefix_table`` (N, pages) int32 -- needed where the first row may have
    nothing mapped.  Rows outside the groups share nothing.  ``kv_last`` (B,)
    int64 is each row's last slot; a row with a negative one (parked) gets zeros.
    All of these are read on the device when the kernels run.  Returns
    (B, KVH, G, 64), written to ``out`` if given.

    It pays for long prefixes or many rows: against each row alone over the shared
    pages (``flash_decode_attention_paged``) 96 rows of a 32768-slot prefix take 36
    us on an MI355X where those take 235, but 4 rows of a 512-slot prefix 9.4 where
    those take 6.3 (14 heads on 2 kv heads; ``PagedDecodeEngine.reads_prefix_once``
    has the rule).
    """
    _half("grouped", grouped, 4)
    b, kvh, g, d = grouped.shape
    index = grouped.get_device()
    pool, cap = _pools(k_pool, v_pool, block_table, b, kvh, index)
    groups = prefix_len.shape[0] if isinstance(prefix_len, torch.Tensor) and prefix_len.dim() == 1 else 0
    if groups < 1:
        raise ValueError("prefix_len must hold at least one group")
    if (_int_rows("prefix_rows", prefix_rows, groups + 1, torch.int32, index) != 1
            or (_int_rows("prefix_len", prefix_len, groups, torch.int32, index) != 1 and groups > 1)):
        raise ValueError("prefix_rows and prefix_len must be contiguous")
    last_sb = _int_rows("kv_last", kv_last, b, torch.int64, index)
    shared = (None, 0, 0)
    if prefix_table is not None:
        if (not isinstance(prefix_table, torch.Tensor) or prefix_table.dtype is not torch.int32
                or prefix_table.get_device() != index):
            raise TypeError(f"prefix_table must be an int32 tensor on cuda:{index}")
        if (prefix_table.dim() != 2 or prefix_table.shape[0] != groups or prefix_table.shape[1] < 1
                or prefix_table.stride(1) != 1):
            raise ValueError(f"prefix_table must be ({groups}, pages >= 1) with unit inner stride")
        shared = (prefix_table.data_ptr(), prefix_table.stride(0), prefix_table.shape[1])
    dev = grouped.device
    if out is None:
        out = (torch.empty_like(grouped) if grouped.is_contiguous()
               else torch.empty((b, kvh, g, d), device=dev, dtype=torch.float16))
    else:
        _half("out", out, 4)
        if out.shape != grouped.shape or out.get_device() != index:
            raise ValueError(f"out must be {tuple(grouped.shape)} on {dev}")
    ws = _workspace(_lib.load().qf_decode_attn_prefix_workspace(b, kvh, g, groups, cap),
                    "qf_decode_attn_prefix_workspace", dev)
    _call("qf_decode_attn_prefix_paged", index, grouped.data_ptr(), *grouped.stride()[:3], *pool,
          prefix_rows.data_ptr(), prefix_len.data_ptr(), groups, *shared, kv_last.data_ptr(), last_sb,
          ws.data_ptr(), ws.shape[0], out.data_ptr(), *out.stride()[:3], b, kvh, g, d,
          d ** -0.5 if scale is None else scale)
    return out


# --------------------------------------------------------------------------
# appends and prefill
# --------------------------------------------------------------------------

def rope_append_paged(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                      cos: torch.Tensor, sin: torch.Tensor, k_pool: torch.Tensor,
                      v_pool: torch.Tensor, block_table: torch.Tensor, slots: torch.Tensor,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """``ops.rope_append`` (SE:927-932) into paged caches at per-row slots.

    query (B, QH, 1, 64), key/value (B, KVH, 1, 64); cos/sin hold B*64 values
    (each row's own position); slots (B,) int64 on the device.  Returns
    rope(query) as (B, QH, 1, 64).
    """
    for n, t in (("query", query), ("key", key), ("value", value)):
        _require_cuda_fp16(n, t, 4)
    b, qh, tq, d = query.shape
    kvh = key.shape[1]
    if tq != 1 or key.shape != (b, kvh, 1, d) or value.shape != key.shape:
        raise ValueError("one token: query (B, QH, 1, D), key/value (B, KVH, 1, D)")
    pool, _ = _pool_args(k_pool, v_pool, block_table, b)
    if k_pool.shape[1] != kvh:
        raise ValueError("pools' kv heads do not match key")
    slot = _slot_args(slots, b, query.device)
    cos2, sin2 = cos.reshape(b, d), sin.reshape(b, d)
    for n, t in (("cos", cos2), ("sin", sin2)):
        if t.dtype != torch.float16 or t.device != query.device or t.stride(1) != 1:
            raise ValueError(f"{n} must be fp16 on the query's device with unit last stride")
    if cos2.stride(0) != sin2.stride(0):
        cos2, sin2 = cos2.contiguous(), sin2.contiguous()
    if out is None:
        out = torch.empty((b, qh, 1, d), device=query.device, dtype=query.dtype)
    with torch.cuda.device(query.device):
        rc = _lib.load().qf_rope_append_paged(
            query.data_ptr(), query.stride(0), query.stride(1),
            key.data_ptr(), key.stride(0), key.stride(1),
            value.data_ptr(), value.stride(0), value.stride(1),
            cos2.data_ptr(), sin2.data_ptr(), cos2.stride(0),
            *pool, *slot, out.data_ptr(), out.stride(0), out.stride(1),
            b, qh, kvh, d, _stream(query.device))
    _lib.check(rc, "qf_rope_append_paged")
    return out


def prefill_varlen_paged(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                         cu_seqlens: torch.Tensor, max_seqlen: int, cos: torch.Tensor | None,
                         sin: torch.Tensor | None, k_pool: torch.Tensor, v_pool: torch.Tensor,
                         block_table: torch.Tensor, start_pos: int = 0,
                         lengths=None) -> torch.Tensor:
    """``ops.prefill_varlen`` appending into paged caches.

    Packed query (T, QH, 64), key/value (T, KVH, 64); cu_seqlens (B+1,) int32
    on the device; optional per-token cos/sin (T, 64).  Token i of row b goes
    to logical slot start_pos + i of row b (start_pos a multiple of 64), then
    each row attends causally over its own tokens.  Returns (T, QH, 64).
    """
    for n, t in (("query", query), ("key", key), ("value", value)):
        _require_cuda_fp16(n, t, 3)
    t_, qh, d = query.shape
    kvh = key.shape[1]
    if key.shape != (t_, kvh, d) or value.shape != key.shape or qh % kvh != 0:
        raise ValueError("packed prefill shapes: query (T, QH, D), key/value (T, KVH, D)")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.device != query.device:
        raise TypeError("cu_seqlens must be a 1-D int32 device tensor")
    b = cu_seqlens.numel() - 1
    if b < 1 or not 1 <= max_seqlen <= t_:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    check_cu_seqlens(cu_seqlens, t_, max_seqlen, lengths)
    if start_pos % 64:
        raise ValueError("start_pos must be a multiple of 64")
    pool, cap = _pool_args(k_pool, v_pool, block_table, b)
    if k_pool.shape[1] != kvh:
        raise ValueError("pools' kv heads do not match key")
    if start_pos + max_seqlen > cap:
        raise ValueError(f"start_pos + max_seqlen exceeds the row capacity {cap}")
    cs_sn = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        for n, t in (("cos", cos), ("sin", sin)):
            _require_cuda_fp16(n, t, 2)
            if t.shape[0] != t_:
                raise ValueError(f"{n} must be (T, 64)")
        if cos.stride(0) != sin.stride(0):
            cos, sin = cos.contiguous(), sin.contiguous()
        cs_sn = cos.stride(0)
    out = torch.empty((t_, qh, d), device=query.device, dtype=torch.float16)
    with torch.cuda.device(query.device):
        rc = _lib.load().qf_prefill_varlen_paged(
            query.data_ptr(), query.stride(1), query.stride(0),
            key.data_ptr(), key.stride(1), key.stride(0),
            value.data_ptr(), value.stride(1), value.stride(0),
            cu_seqlens.data_ptr(), t_, int(max_seqlen),
            _ptr(cos), _ptr(sin), cs_sn,
            *pool, int(start_pos),
            out.data_ptr(), out.stride(1), out.stride(0),
            b, qh, kvh, d, float(d ** -0.5), _stream(query.device))
    _lib.check(rc, "qf_prefill_varlen_paged")
    return out


def prefill_extend_paged(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                         cu_seqlens: torch.Tensor, max_seqlen: int, context: torch.Tensor,
                         cos: torch.Tensor | None, sin: torch.Tensor | None, k_pool: torch.Tensor,
                         v_pool: torch.Tensor, block_table: torch.Tensor, lengths=None,
                         max_slots: int | None = None, scale: float | None = None) -> torch.Tensor:
    """``prefill_varlen_paged`` for rows that hold slots already.

    Packed query (T, QH, 64), key/value (T, KVH, 64) of the rows' new tokens;
    row b's token i goes to its slot context[b] + i and attends to slots
    [0, context[b] + i].  ``cu_seqlens``, ``max_seqlen`` and ``lengths`` as
    there, but a row may have no tokens.  ``context`` (B,) int64 is read on the
    device; a row with a negative one appends nothing and gets zeros.
    ``cos``/``sin`` (T, 64) are the tokens' own tables, or None for q and k that
    are rotated already.  ``max_slots`` bounds every row's context + tokens
    (default: the table's): the work is split by it, and slots past it are
    neither written nor read.  Pages that hold the new slots must be the row's
    own (``PagedKvCache.own_slots``).  Returns (T, QH, 64).
    """
    _half("query", query, 3)
    _half("key", key, 3)
    _half("value", value, 3)
    t_, qh, d = query.shape
    kvh = key.shape[1]
    if key.shape[0] != t_ or value.shape != key.shape or kvh < 1 or qh % kvh != 0:
        raise ValueError("packed extension shapes: query (T, QH, D), key/value (T, KVH, D)")
    index, dev = query.get_device(), query.device
    if key.get_device() != index or value.get_device() != index:
        raise ValueError(f"query, key and value must be on one device ({dev})")
    b = cu_seqlens.shape[0] - 1 if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.dim() == 1 else 0
    if b < 1 or not 1 <= max_seqlen <= t_:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    if _int_rows("cu_seqlens", cu_seqlens, b + 1, torch.int32, index) != 1:
        raise ValueError("cu_seqlens must be contiguous")
    ctx_sb = _int_rows("context", context, b, torch.int64, index)
    _check_rows(cu_seqlens, t_, max_seqlen, lengths)
    pool, cap = _pools(k_pool, v_pool, block_table, b, kvh, index)
    if max_slots is not None:
        if not max_seqlen <= max_slots <= cap:
            raise ValueError(f"max_slots must be in [{max_seqlen}, {cap}] (got {max_slots})")
        cap = int(max_slots)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    cs_sn = 0
    if cos is not None:
        for n, t in (("cos", cos), ("sin", sin)):
            _half(n, t, 2)
            if t.shape[0] != t_ or t.get_device() != index:
                raise ValueError(f"{n} must be (T, 64) on {dev}")
        if cos.stride(0) != sin.stride(0):
            cos, sin = cos.contiguous(), sin.contiguous()
        cs_sn = cos.stride(0)
    out = torch.empty((t_, qh, d), device=dev, dtype=torch.float16)
    ws = _workspace(_lib.load().qf_prefill_extend_workspace(b, qh, kvh, t_, cap),
                    "qf_prefill_extend_workspace", dev)
    qs, ks, vs = query.stride(), key.stride(), value.stride()
    _call("qf_prefill_extend_paged", index, query.data_ptr(), qs[1], qs[0], key.data_ptr(), ks[1], ks[0],
          value.data_ptr(), vs[1], vs[0], cu_seqlens.data_ptr(), t_, context.data_ptr(), ctx_sb, _ptr(cos),
          _ptr(sin), cs_sn, *pool, cap, ws.data_ptr(), ws.shape[0], out.data_ptr(), d, qh * d, b, qh, kvh, d,
          d ** -0.5 if scale is None else scale)
    return out


def rms_qkv_rope_append_paged(x: torch.Tensor, norm_w: torch.Tensor, eps: float,
                              w_qkv, bias: torch.Tensor | None,
                              cos: torch.Tensor | None, sin: torch.Tensor | None,
                              k_pool: torch.Tensor, v_pool: torch.Tensor,
                              block_table: torch.Tensor, slots: torch.Tensor,
                              q_out: torch.Tensor, token: torch.Tensor | None = None,
                              hidden_out: torch.Tensor | None = None, positions=None) -> None:
    """``step_ops.rms_qkv_rope_append`` appending into paged caches at per-row
    ``slots`` (B,) int64; RoPE from cos/sin tables or ``positions =
    (pos, inv_freq)`` as there."""
    _check("q_out", q_out)
    if q_out.dim() != 3 or q_out.shape[2] != HEAD_DIM or q_out.stride(2) != 1:
        raise ValueError(f"q_out must be (B, QH, 64) (got {tuple(q_out.shape)})")
    b, qh = q_out.shape[0], q_out.shape[1]
    _batch(b)
    pool, _ = _pool_args(k_pool, v_pool, block_table, b)
    kvh = k_pool.shape[1]
    hidden = norm_w.shape[0]
    _check("norm_w", norm_w)
    w_ptr, w_layout = _weight("w_qkv", w_qkv, (qh + 2 * kvh) * HEAD_DIM, hidden, PACK_ROPE)
    if bias is not None:
        _check("bias", bias)
        if tuple(bias.shape) != ((qh + 2 * kvh) * HEAD_DIM,) or not bias.is_contiguous():
            raise ValueError("bias must be contiguous ((QH + 2 KVH) * 64,)")
    rope = rope_args(cos, sin, positions, b)
    slot = _slot_args(slots, b, q_out.device)
    if token is not None:
        _check("token", token, torch.int64)
        if token.shape != (b,) or not token.is_contiguous():
            raise ValueError("token must be contiguous (B,)")
        _check("x", x)
        if x.dim() != 2 or x.shape[1] != hidden or x.stride(1) != 1:
            raise ValueError("embedding table must be (vocab, hidden)")
        x_sb = x.stride(0)
        ho_sb = _rows("hidden_out", hidden_out, b, hidden) if hidden_out is not None else 0
    else:
        x_sb = _rows("x", x, b, hidden)
        ho_sb = 0
        hidden_out = None
    rc = _lib.load().qf_rms_qkv_rope_append_paged(
        x.data_ptr(), x_sb, _ptr(token), _ptr(hidden_out), ho_sb,
        norm_w.data_ptr(), float(eps), w_ptr, w_layout, _ptr(bias), *rope, *pool, *slot,
        q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
        b, hidden, qh, kvh, HEAD_DIM, _stream(x.device))
    _lib.check(rc, "qf_rms_qkv_rope_append_paged")
