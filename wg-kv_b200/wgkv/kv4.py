"""A paged KV cache held in 4 bits: written, read back and attended.

``paged_decode`` is bound by the bytes of K and V it reads; a 4-bit cache has 3.2 to 3.8 times fewer.
A value is ``scale * code + minimum`` with a bf16 (minimum, scale) pair for every ``group_size``
consecutive dimensions of one token's K or V row (the exact rule is stated at ``wgkv_kv4_row_bytes`` in
include/wgkv.h).  The cache is one tensor ``(num_pages, page_size, row_bytes)`` uint8, addressed like the
bf16 pages of :func:`wgkv.paged_decode`: ``block_table[b, h]`` lists the pages of a head, logical position
``p`` lives in page ``p // page_size``.  ``row_bytes`` tells head size and group size apart, so no call
takes them.

* :func:`kv4_alloc` -- an empty cache;
* :func:`kv4_append` -- quantise K/V rows as they are written at each head's own position (prompt chunks
  and single decode tokens alike);
* :func:`kv4_read` -- rows back as bf16;
* :func:`paged_decode_kv4` -- one query token per sequence over the cache.

None of them synchronises; positions past a head's table and page ids outside the cache are reported
through ``wgkv.check_errors()``.  The pool uses the same cache when ``init_pool`` is given ``kv_group``.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .runtime import err_word, require_cuda, stream_ptr, workspace

GROUPS = {64: (32, 64), 128: (32, 64, 128)}  # head size -> group sizes
_BY_ROW = {d + 8 * (d // g): (d, g) for d, gs in GROUPS.items() for g in gs}


def kv4_row_bytes(head_dim, group_size=64):
    """Bytes of one token's K and V in a 4-bit cache."""
    if group_size not in GROUPS.get(head_dim, ()):
        raise ValueError(f"a 4-bit cache needs head_dim 64 (groups 32, 64) or 128 (groups 32, 64, 128), "
                         f"got head_dim {head_dim}, group_size {group_size}")
    return head_dim + 8 * (head_dim // group_size)


def kv4_alloc(num_pages, page_size, head_dim, group_size=64, device="cuda"):
    """An empty 4-bit cache: (num_pages, page_size, row_bytes) uint8, every value 0."""
    if num_pages <= 0 or page_size <= 0 or page_size % 16:
        raise ValueError(f"num_pages must be positive and page_size a multiple of 16, got {num_pages}, {page_size}")
    return torch.zeros(num_pages, page_size, kv4_row_bytes(head_dim, group_size), dtype=torch.uint8, device=device)


def _cache_dims(cache):
    """(head size, group size) of a cache tensor."""
    if cache.dtype != torch.uint8:
        raise TypeError(f"a 4-bit cache is a uint8 tensor, got {cache.dtype}")
    if cache.dim() != 3 or cache.shape[2] not in _BY_ROW or cache.shape[0] == 0 or cache.shape[1] == 0 or \
            cache.shape[1] % 16:
        raise ValueError(f"a 4-bit cache is (num_pages, page_size, row_bytes) with page_size a multiple of 16 and "
                         f"row_bytes one of {sorted(_BY_ROW)}, got {tuple(cache.shape)}")
    if not cache.is_contiguous():
        raise ValueError("a 4-bit cache must be contiguous")
    return _BY_ROW[cache.shape[2]]


def _heads(t, name, B, Hk, dev):
    """A (B, Hk) int32 tensor."""
    if t.shape != (B, Hk):
        raise ValueError(f"{name} must be (B, Hk) = ({B}, {Hk}), got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
    if t.dtype != torch.int32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise TypeError(f"{name} must hold integers, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _table(t, dev):
    """The block table (B, Hk, n) as int32 rows and their distance in elements."""
    if t.dim() != 3 or t.numel() == 0:
        raise ValueError(f"block_table must be (B, Hk, pages), none of them 0, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"block_table is on {t.device}, the cache on {dev}")
    if t.dtype != torch.int32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise TypeError(f"block_table must hold integers, got {t.dtype}")
        t = t.to(torch.int32)
    B, Hk, w = t.shape
    rows = t.stride(1) if Hk > 1 else t.stride(0) if B > 1 else w
    if (w > 1 and t.stride(2) != 1) or rows < w or (B > 1 and Hk > 1 and t.stride(0) != Hk * rows):
        t, rows = t.contiguous(), w
    return t, rows


def _check_call(status, what, B, Hk, width, cache):
    if status == -1:
        if cache.data_ptr() % 16:
            raise ValueError(f"{what}: the cache is not 16-byte aligned")
        raise ValueError(f"{what}: refused sizes (B {B}, Hk {Hk}, table of {width} pages of {cache.shape[1]} tokens)")
    check(status, what)


class _on:
    """The tensors' device as the current one (a no-op where it is already)."""
    __slots__ = ("guard",)

    def __init__(self, dev):
        self.guard = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def kv4_append(k, v, cache, start, block_table, counts=None):
    """Quantise rows into ``cache``: row r of (b, h) to logical position ``start[b, h] + r``.

    k, v (B, Hk, L, D) bf16, any strides with a contiguous last axis (others are copied first); start and
    counts (B, Hk) integers; rows ``r >= counts[b, h]`` are skipped (``counts=None``: none are).  Only the
    rows written change.  Rows past the head's table are dropped and reported by ``check_errors()``; no
    two rows of one call may name the same place.  Returns ``cache``."""
    for t, n in ((k, "k"), (v, "v"), (cache, "cache"), (start, "start"), (block_table, "block_table")):
        require_cuda(t, n)
    D, group = _cache_dims(cache)
    dev = cache.device
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError(f"k and v must be bf16, got {k.dtype} and {v.dtype}")
    if k.dim() != 4 or k.shape != v.shape or k.shape[3] != D:
        raise ValueError(f"k and v must be (B, Hk, L, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.device != dev or v.device != dev:
        raise ValueError(f"k is on {k.device}, v on {v.device}, the cache on {dev}")
    B, Hk, L, _ = k.shape
    if block_table.shape[:2] != (B, Hk):
        raise ValueError(f"block_table must be ({B}, {Hk}, pages), got {tuple(block_table.shape)}")
    start = _heads(start, "start", B, Hk, dev)
    if counts is not None:
        require_cuda(counts, "counts")
        counts = _heads(counts, "counts", B, Hk, dev)
    bt, bt_rows = _table(block_table, dev)
    if L == 0:
        return cache
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    with _on(dev):
        st = lib.wgkv_kv4_append(k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0),
                                 v.stride(1), v.stride(2), B, Hk, L, D, group, cache.data_ptr(), cache.shape[0],
                                 cache.shape[1], start.data_ptr(), counts.data_ptr() if counts is not None else None,
                                 bt.data_ptr(), bt_rows, bt.shape[2], err_word(dev).data_ptr(), stream_ptr(dev))
    _check_call(st, "wgkv_kv4_append", B, Hk, bt.shape[2], cache)
    return cache


def kv4_read(cache, start, counts, block_table, max_rows, out=None):
    """Rows of ``cache`` back as bf16: (k, v), each (B, Hk, max_rows, D).

    Row i of (b, h) is logical position ``start[b, h] + i`` (``start=None``: i) for
    ``i < min(counts[b, h], max_rows)`` and zero behind that.  ``out``: two contiguous bf16 tensors to
    fill."""
    for t, n in ((cache, "cache"), (counts, "counts"), (block_table, "block_table")):
        require_cuda(t, n)
    D, group = _cache_dims(cache)
    dev = cache.device
    bt, bt_rows = _table(block_table, dev)
    B, Hk, width = bt.shape
    counts = _heads(counts, "counts", B, Hk, dev)
    if start is not None:
        require_cuda(start, "start")
        start = _heads(start, "start", B, Hk, dev)
    max_rows = int(max_rows)
    if max_rows < 0:
        raise ValueError(f"max_rows must not be negative, got {max_rows}")
    shape = (B, Hk, max_rows, D)
    if out is None:
        ok, ov = (torch.empty(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
    else:
        ok, ov = out
        for t in (ok, ov):
            if t.dtype != torch.bfloat16 or t.shape != shape or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"out must be two contiguous bf16 tensors {shape} on {dev}")
    if max_rows == 0:
        return ok, ov
    if (ok.data_ptr() | ov.data_ptr()) % 16:
        raise ValueError("out must be 16-byte aligned")
    with _on(dev):
        st = lib.wgkv_kv4_read(cache.data_ptr(), cache.shape[0], cache.shape[1], D, group,
                               start.data_ptr() if start is not None else None, counts.data_ptr(), bt.data_ptr(),
                               bt_rows, width, B, Hk, max_rows, ok.data_ptr(), ov.data_ptr(),
                               err_word(dev).data_ptr(), stream_ptr(dev))
    _check_call(st, "wgkv_kv4_read", B, Hk, width, cache)
    return ok, ov


def _decode_args(q, cache, cache_seqlens, block_table):
    D, group = _cache_dims(cache)
    dev = cache.device
    if q.dtype != torch.bfloat16:
        raise TypeError(f"q must be bf16, got {q.dtype}")
    if q.dim() != 4 or q.shape[1] != 1 or q.shape[3] != D:
        raise ValueError(f"q must be (B, 1, Hq, {D}), got {tuple(q.shape)}")
    if q.device != dev:
        raise ValueError(f"q is on {q.device}, the cache on {dev}")
    B, Hq = q.shape[0], q.shape[2]
    if block_table.dim() != 3 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be (B, Hk, pages) with B = {B}, got {tuple(block_table.shape)}")
    Hk = block_table.shape[1]
    if Hk == 0 or Hq == 0 or Hq % Hk or Hq // Hk > 16:
        raise ValueError(f"query heads ({Hq}) must be 1 to 16 times the KV heads ({Hk})")
    return B, Hq, Hk, D, group, dev


def paged_decode_kv4(q, cache, cache_seqlens, block_table, softmax_scale, out=None):
    """out (B, 1, Hq, D) bf16 = GQA softmax attention of q over the first ``cache_seqlens[b, h]`` positions
    of each head's pages in a 4-bit cache (:func:`wgkv.paged_decode` for such a cache).

    A head of length 0 gives zeros.  A length past the table's pages is cut there and reported by
    ``check_errors()``.  Hq / Hk at most 16; any B * Hk up to 4096."""
    for t, n in ((q, "q"), (cache, "cache"), (cache_seqlens, "cache_seqlens"), (block_table, "block_table")):
        require_cuda(t, n)
    B, Hq, Hk, D, group, dev = _decode_args(q, cache, cache_seqlens, block_table)
    sl = _heads(cache_seqlens, "cache_seqlens", B, Hk, dev)
    bt, bt_rows = _table(block_table, dev)
    if not q.is_contiguous():
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be contiguous and like q")
    elif out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    if q.data_ptr() % 16:
        q = q.clone()
    with _on(dev):
        nbytes = int(lib.wgkv_paged_decode_kv4_workspace_size(B, Hq, Hk, D))
        counters = ((B * Hk * 4 + 255) // 256) * 256
        if torch.cuda.is_current_stream_capturing():
            # a graph's own scratch (from its memory pool): graphs captured on one stream may replay on
            # several, and must then not share the partial results and counters of the stream's scratch
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ws[:counters].zero_()
        else:
            ws = workspace(dev, "paged_decode_kv4", nbytes, zero_prefix=counters)
        st = lib.wgkv_paged_decode_kv4(q.data_ptr(), cache.data_ptr(), cache.shape[0], cache.shape[1], group,
                                       sl.data_ptr(), bt.data_ptr(), bt_rows, bt.shape[2], B, Hq, Hk, D,
                                       float(softmax_scale), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                       err_word(dev).data_ptr(), stream_ptr(dev))
    _check_call(st, "wgkv_paged_decode_kv4", B, Hk, bt.shape[2], cache)
    return out
