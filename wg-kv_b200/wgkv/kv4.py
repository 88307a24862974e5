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

import struct

import torch

from ._lib import check, lib
from .runtime import counter_scratch, err_word, raw_stream, require_cuda

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


# wgkv_kv4_call's operations and the formats of their slots: the host's share of a small call is of the
# order of the kernel, and converting 20 arguments one by one through ctypes is half of it
_APPEND, _READ, _DECODE = 0, 1, 2
_APPEND_SLOTS, _READ_SLOTS, _DECODE_SLOTS = struct.Struct("=23q"), struct.Struct("=17q"), struct.Struct("=13qd5q")
# What a call's shapes say, checked once for each combination of them: (tensor shapes) -> sizes
_append_plans: dict = {}
_read_plans: dict = {}
_decode_plans: dict = {}
_scratch: dict = {}   # (device index, B, Hq, Hk, D) -> workspace bytes of paged_decode_kv4
_err_ptrs: dict = {}  # device index -> (address of its error word, the word)
_BF16, _I32 = torch.bfloat16, torch.int32
_COUNTER_BYTES = 32768  # of paged_decode_kv4's workspace, zero between calls


def _remember(plans, key, plan):
    if len(plans) >= 4096:  # shapes that change with every call
        plans.clear()
    plans[key] = plan
    return plan


def _cache_dims(cache):
    """(head size, group size) of a cache tensor."""
    if cache.dtype is torch.uint8 and cache.dim() == 3:
        n, page, row = cache.shape
        dims = _BY_ROW.get(row)
        if dims is not None and n and page and page % 16 == 0:
            if not cache.is_contiguous():
                raise ValueError("a 4-bit cache must be contiguous")
            return dims
    if cache.dtype != torch.uint8:
        raise TypeError(f"a 4-bit cache is a uint8 tensor, got {cache.dtype}")
    raise ValueError(f"a 4-bit cache is (num_pages, page_size, row_bytes) with page_size a multiple of 16 and "
                     f"row_bytes one of {sorted(_BY_ROW)}, got {tuple(cache.shape)}")


def _refuse_devices(cache, **tensors):
    """Says which of the tensors is not on the cache's GPU."""
    require_cuda(cache, "cache")
    for name, t in tensors.items():
        if t is not None:
            require_cuda(t, name)
            if t.get_device() != cache.get_device():
                raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")


def _integers(t, name):
    if t.dtype is not _I32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype is torch.bool:
            raise TypeError(f"{name} must hold integers, got {t.dtype}")
        if t.dtype is torch.int64:  # out of range stays out of range
            t = t.clamp(-2 ** 31, 2 ** 31 - 1)
        t = t.to(_I32)
    return t


def _check_heads(shape, name, B, Hk):
    if tuple(shape) != (B, Hk):
        raise ValueError(f"{name} must be (B, Hk) = ({B}, {Hk}), got {tuple(shape)}")


def _heads(t, name):
    """A (B, Hk) tensor as contiguous int32."""
    t = _integers(t, name)
    return t if t.is_contiguous() else t.contiguous()


def _table_dims(shape):
    if len(shape) != 3 or 0 in shape:
        raise ValueError(f"block_table must be (B, Hk, pages), none of them 0, got {tuple(shape)}")
    return shape


def _table(t):
    """The block table (B, Hk, n) as int32 rows, and their distance in elements."""
    t = _integers(t, "block_table")
    B, Hk, w = t.shape
    if t.is_contiguous():
        return t, w
    rows = t.stride(1) if Hk > 1 else t.stride(0) if B > 1 else w
    if (w > 1 and t.stride(2) != 1) or rows < w or (B > 1 and Hk > 1 and t.stride(0) != Hk * rows):
        t, rows = t.contiguous(), w
    return t, rows


def _call(index, op, slots, what, B, Hk, width, cache):
    status = lib.wgkv_kv4_call(op, slots)
    if status:
        if status == -1:
            if cache.data_ptr() % 16:
                raise ValueError(f"{what}: the cache is not 16-byte aligned")
            raise ValueError(f"{what}: refused sizes (B {B}, Hk {Hk}, table of {width} pages of {cache.shape[1]} "
                             f"tokens, {cache.shape[0]} pages in the cache)")
        check(status, what)


def _err_ptr(index):
    p = _err_ptrs.get(index)
    if p is None:
        word = err_word(torch.device("cuda", index))
        p = _err_ptrs[index] = word.data_ptr(), word
    return p[0]


def _append_plan(k, v, cache, start, block_table, counts):
    D, group = _cache_dims(cache)
    B, Hk, width = _table_dims(block_table.shape)
    if k.dim() != 4 or k.shape != v.shape or k.shape[3] != D or k.shape[0] != B or k.shape[1] != Hk:
        raise ValueError(f"k and v must be ({B}, {Hk}, L, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    _check_heads(start.shape, "start", B, Hk)
    if counts is not None:
        _check_heads(counts.shape, "counts", B, Hk)
    return B, Hk, k.shape[2], D, group, cache.shape[0], cache.shape[1], width


def kv4_append(k, v, cache, start, block_table, counts=None):
    """Quantise rows into ``cache``: row r of (b, h) to logical position ``start[b, h] + r``.

    k, v (B, Hk, L, D) bf16, any strides with a contiguous last axis (others are copied first); start and
    counts (B, Hk) integers; rows ``r >= counts[b, h]`` are skipped (``counts=None``: none are).  Only the
    rows written change.  Rows past the head's table are dropped and reported by ``check_errors()``; no
    two rows of one call may name the same place.  Returns ``cache``."""
    index = cache.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index or start.get_device() != index or \
            block_table.get_device() != index or (counts is not None and counts.get_device() != index):
        _refuse_devices(cache, k=k, v=v, start=start, block_table=block_table, counts=counts)
    if k.dtype is not _BF16 or v.dtype is not _BF16:
        raise TypeError(f"k and v must be bf16, got {k.dtype} and {v.dtype}")
    key = (k.shape, v.shape, cache.shape, start.shape, block_table.shape, counts.shape if counts is not None else None)
    plan = _append_plans.get(key)
    if plan is None or cache.dtype is not torch.uint8 or not cache.is_contiguous():
        plan = _remember(_append_plans, key, _append_plan(k, v, cache, start, block_table, counts))
    B, Hk, L, D, group, pages, page, width = plan
    start = _heads(start, "start")
    counts_ptr = 0
    if counts is not None:
        counts = _heads(counts, "counts")
        counts_ptr = counts.data_ptr()
    bt, bt_rows = _table(block_table)
    if L == 0:
        return cache
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return kv4_append(k, v, cache, start, bt, counts)
    k_sb, k_sh, k_st, k_sd = k.stride()
    v_sb, v_sh, v_st, v_sd = v.stride()
    if k_sd != 1:
        k = k.contiguous()
        k_sb, k_sh, k_st, _ = k.stride()
    if v_sd != 1:
        v = v.contiguous()
        v_sb, v_sh, v_st, _ = v.stride()
    _call(index, _APPEND,
          _APPEND_SLOTS.pack(k.data_ptr(), k_sb, k_sh, k_st, v.data_ptr(), v_sb, v_sh, v_st, B, Hk, L, D, group,
                             cache.data_ptr(), pages, page, start.data_ptr(), counts_ptr, bt.data_ptr(), bt_rows, width,
                             _err_ptr(index), raw_stream(index)), "wgkv_kv4_append", B, Hk, width, cache)
    return cache


def _read_plan(cache, start, counts, block_table, max_rows):
    D, group = _cache_dims(cache)
    B, Hk, width = _table_dims(block_table.shape)
    _check_heads(counts.shape, "counts", B, Hk)
    if start is not None:
        _check_heads(start.shape, "start", B, Hk)
    if max_rows < 0:
        raise ValueError(f"max_rows must not be negative, got {max_rows}")
    return B, Hk, D, group, cache.shape[0], cache.shape[1], width, (B, Hk, max_rows, D)


def kv4_read(cache, start, counts, block_table, max_rows, out=None):
    """Rows of ``cache`` back as bf16: (k, v), each (B, Hk, max_rows, D).

    Row i of (b, h) is logical position ``start[b, h] + i`` (``start=None``: i) for
    ``i < min(counts[b, h], max_rows)`` and zero behind that.  ``out``: two contiguous bf16 tensors to
    fill."""
    index = cache.get_device()
    if index < 0 or counts.get_device() != index or block_table.get_device() != index or \
            (start is not None and start.get_device() != index):
        _refuse_devices(cache, counts=counts, block_table=block_table, start=start)
    max_rows = int(max_rows)
    key = (cache.shape, counts.shape, block_table.shape, max_rows, start.shape if start is not None else None)
    plan = _read_plans.get(key)
    if plan is None or cache.dtype is not torch.uint8 or not cache.is_contiguous():
        plan = _remember(_read_plans, key, _read_plan(cache, start, counts, block_table, max_rows))
    B, Hk, D, group, pages, page, width, shape = plan
    bt, bt_rows = _table(block_table)
    counts = _heads(counts, "counts")
    start_ptr = 0
    if start is not None:
        start = _heads(start, "start")
        start_ptr = start.data_ptr()
    if out is None:
        ok = cache.new_empty(shape, dtype=_BF16)
        ov = torch.empty_like(ok)
    else:
        ok, ov = out
        for t in (ok, ov):
            if t.dtype is not _BF16 or t.shape != shape or not t.is_contiguous() or t.get_device() != index:
                raise ValueError(f"out must be two contiguous bf16 tensors {shape} on {cache.device}")
    if max_rows == 0:
        return ok, ov
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return kv4_read(cache, start, counts, bt, max_rows, (ok, ov))
    k_ptr, v_ptr = ok.data_ptr(), ov.data_ptr()
    if (k_ptr | v_ptr) % 16:
        raise ValueError("out must be 16-byte aligned")
    _call(index, _READ,
          _READ_SLOTS.pack(cache.data_ptr(), pages, page, D, group, start_ptr, counts.data_ptr(), bt.data_ptr(), bt_rows,
                           width, B, Hk, max_rows, k_ptr, v_ptr, _err_ptr(index), raw_stream(index)), "wgkv_kv4_read",
          B, Hk, width, cache)
    return ok, ov


def _decode_plan(q, cache, cache_seqlens, block_table):
    D, group = _cache_dims(cache)
    B, Hk, width = _table_dims(block_table.shape)
    if q.dim() != 4 or q.shape[0] != B or q.shape[1] != 1 or q.shape[3] != D:
        raise ValueError(f"q must be ({B}, 1, Hq, {D}), got {tuple(q.shape)}")
    Hq = q.shape[2]
    if Hq == 0 or Hq % Hk or Hq > 16 * Hk:
        raise ValueError(f"query heads ({Hq}) must be 1 to 16 times the KV heads ({Hk})")
    _check_heads(cache_seqlens.shape, "cache_seqlens", B, Hk)
    return B, Hq, Hk, D, group, cache.shape[0], cache.shape[1], width


def paged_decode_kv4(q, cache, cache_seqlens, block_table, softmax_scale, out=None):
    """out (B, 1, Hq, D) bf16 = GQA softmax attention of q over the first ``cache_seqlens[b, h]`` positions
    of each head's pages in a 4-bit cache (:func:`wgkv.paged_decode` for such a cache).

    A head of length 0 gives zeros.  A length past the table's pages is cut there and reported by
    ``check_errors()``.  Hq / Hk at most 16; any B * Hk up to 4096."""
    index = cache.get_device()
    if index < 0 or q.get_device() != index or cache_seqlens.get_device() != index or block_table.get_device() != index:
        _refuse_devices(cache, q=q, cache_seqlens=cache_seqlens, block_table=block_table)
    if q.dtype is not _BF16:
        raise TypeError(f"q must be bf16, got {q.dtype}")
    key = (q.shape, cache.shape, cache_seqlens.shape, block_table.shape)
    plan = _decode_plans.get(key)
    if plan is None or cache.dtype is not torch.uint8 or not cache.is_contiguous():
        plan = _remember(_decode_plans, key, _decode_plan(q, cache, cache_seqlens, block_table))
    B, Hq, Hk, D, group, pages, page, width = plan
    sl = _heads(cache_seqlens, "cache_seqlens")
    bt, bt_rows = _table(block_table)
    if not q.is_contiguous():
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype is not _BF16 or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index:
        raise ValueError("out must be contiguous and like q")
    elif out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return paged_decode_kv4(q, cache, sl, bt, softmax_scale, out)
    q_ptr = q.data_ptr()
    if q_ptr % 16:
        q = q.clone()
        q_ptr = q.data_ptr()
    heads = (index, B, Hq, Hk, D)
    need = _scratch.get(heads)
    if need is None:
        need = _remember(_scratch, heads, int(lib.wgkv_paged_decode_kv4_workspace_size(B, Hq, Hk, D)))
    stream = raw_stream(index)
    ws, ws_bytes = counter_scratch(index, stream, "paged_decode_kv4", need, _COUNTER_BYTES)
    _call(index, _DECODE,
          _DECODE_SLOTS.pack(q_ptr, cache.data_ptr(), pages, page, group, sl.data_ptr(), bt.data_ptr(), bt_rows, width,
                             B, Hq, Hk, D, softmax_scale, out.data_ptr(), ws, ws_bytes, _err_ptr(index), stream),
          "wgkv_paged_decode_kv4", B, Hk, width, cache)
    return out
