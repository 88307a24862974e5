"""The 4-bit KV cache without a GPU: sizes, refusals of the C entry points and of the Python calls, shape
propagation of the registered operators, and the oracle's own rule and layout."""
import os

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import wgkv
import wgkv.ops  # noqa: F401
from oracle import kv4_oracle as K4
from wgkv._lib import LIB_PATH, lib

EINVAL, ENOSPC = -1, -3
COMBOS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]
needs_lib = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="libwgkv.so not built")


@needs_lib
def test_row_bytes():
    for D in (32, 64, 96, 128, 256):
        for g in (16, 32, 64, 128, 256):
            if (D, g) in COMBOS:
                assert lib.wgkv_kv4_row_bytes(D, g) == wgkv.kv4_row_bytes(D, g) == D + 8 * D // g
            else:
                assert lib.wgkv_kv4_row_bytes(D, g) == EINVAL
                with pytest.raises(ValueError):
                    wgkv.kv4_row_bytes(D, g)
    assert len({wgkv.kv4_row_bytes(*c) for c in COMBOS}) == len(COMBOS)  # a row size names its combination


F = 4096  # non-null, 16-byte aligned, never touched


def _append(k=F, v=F, B=1, Hk=2, L=3, D=128, g=64, cache=F, pages=8, page=16, start=F, counts=None, table=F, stride=4,
            width=4):
    return lib.wgkv_kv4_append(k, 8, 8, 8, v, 8, 8, 8, B, Hk, L, D, g, cache, pages, page, start, counts, table,
                               stride, width, F, None)


def _read(cache=F, pages=8, page=16, D=128, g=64, counts=F, table=F, stride=4, width=4, B=1, Hk=2, rows=3, k=F, v=F):
    return lib.wgkv_kv4_read(cache, pages, page, D, g, None, counts, table, stride, width, B, Hk, rows, k, v, F, None)


def _decode(q=F, cache=F, pages=8, page=16, g=64, sl=F, table=F, stride=4, width=4, B=1, Hq=8, Hk=2, D=128, out=F,
            ws=F, nbytes=1 << 30):
    return lib.wgkv_paged_decode_kv4(q, cache, pages, page, g, sl, table, stride, width, B, Hq, Hk, D, 1.0, out, ws,
                                     nbytes, F, None)


@needs_lib
@pytest.mark.parametrize("call", [_append, _read, _decode])
def test_entry_points_refuse_before_any_device_work(call):
    big = 1 << 28
    for bad in (dict(D=96), dict(D=64, g=128), dict(g=16), dict(cache=None), dict(cache=F + 8), dict(pages=0),
                dict(page=24), dict(page=0), dict(table=None), dict(width=0), dict(stride=3), dict(B=0), dict(Hk=0),
                dict(B=65536), dict(width=big, stride=big)):
        assert call(**bad) == EINVAL, bad


@needs_lib
def test_entry_points_refuse_what_is_theirs():
    for bad in (dict(k=None), dict(v=None), dict(start=None), dict(L=-1)):
        assert _append(**bad) == EINVAL, bad
    for bad in (dict(counts=None), dict(k=None), dict(v=None), dict(k=F + 2), dict(v=F + 8), dict(rows=-1)):
        assert _read(**bad) == EINVAL, bad
    for bad in (dict(q=None), dict(q=F + 2), dict(sl=None), dict(out=None), dict(out=F + 8), dict(ws=None),
                dict(Hq=7), dict(Hq=0), dict(Hq=34), dict(B=2049)):
        assert _decode(**bad) == EINVAL, bad
    # records of 16 tokens are counted in 32 bits over all heads
    assert _decode(B=1024, Hk=4, Hq=8, width=1 << 20, stride=1 << 20, page=64) == EINVAL
    assert _decode(nbytes=0) == ENOSPC
    assert _append(L=0) == 0 and _read(rows=0) == 0  # nothing to do, nothing launched


def _t(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def test_python_calls_refuse_cpu_tensors():
    c = torch.zeros(4, 16, 144, dtype=torch.uint8)
    k = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    n, bt = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        wgkv.kv4_append(k, k, c, n, bt)
    with pytest.raises(RuntimeError):
        wgkv.kv4_read(c, None, n, bt, 3)
    with pytest.raises(RuntimeError):
        wgkv.paged_decode_kv4(k[:, :1], c, n, bt, 1.0)
    with pytest.raises(NotImplementedError):
        torch.ops.wgkv.paged_decode_kv4(k[:, :1], c, n, bt, 1.0)


def test_python_calls_refuse_bad_arguments():
    with FakeTensorMode():
        c, bt, n = _t(9, 16, 144, dtype=torch.uint8), _i(2, 3, 4), _i(2, 3)
        k, q = _t(2, 3, 5, 128), _t(2, 1, 6, 128)
        bad_caches = [(_t(9, 16, 143, dtype=torch.uint8), ValueError), (_t(9, 24, 144, dtype=torch.uint8), ValueError),
                      (_t(0, 16, 144, dtype=torch.uint8), ValueError), (_t(9, 16 * 144, dtype=torch.uint8), ValueError),
                      (_t(9, 16, 144), TypeError), (_t(9, 32, 144, dtype=torch.uint8)[:, ::2], ValueError)]
        for x, e in bad_caches:
            for f in (lambda: wgkv.kv4_append(k, k, x, n, bt), lambda: wgkv.kv4_read(x, None, n, bt, 5),
                      lambda: wgkv.paged_decode_kv4(q, x, n, bt, 1.0)):
                with pytest.raises(e):
                    f()
        for args, e in [((_t(2, 3, 5, 64), _t(2, 3, 5, 64), c, n, bt), ValueError),  # head size of the cache: 128
                        ((k, _t(2, 3, 4, 128), c, n, bt), ValueError),
                        ((k.float(), k, c, n, bt), TypeError),
                        ((k, k.half(), c, n, bt), TypeError),
                        ((k, k, c, _i(3, 2), bt), ValueError),
                        ((k, k, c, _t(2, 3), bt), TypeError),
                        ((k, k, c, n, _i(2, 2, 4)), ValueError),
                        ((k, k, c, n, _i(2, 3, 0)), ValueError),
                        ((k, k, c, n, _t(2, 3, 4)), TypeError),
                        ((k, k, c, n, bt, _i(2, 2)), ValueError)]:
            with pytest.raises(e):
                wgkv.kv4_append(*args)
        for args, e in [((c, None, _i(2, 2), bt, 5), ValueError), ((c, _i(3, 3), n, bt, 5), ValueError),
                        ((c, None, n, bt, -1), ValueError), ((c, None, n, _i(6, 4), 5), ValueError),
                        ((c, None, n, bt, 5, (_t(2, 3, 5, 128), _t(2, 3, 4, 128))), ValueError)]:
            with pytest.raises(e):
                wgkv.kv4_read(*args)
        for args, e in [((_t(2, 2, 6, 128), c, n, bt, 1.0), ValueError), ((_t(2, 1, 7, 128), c, n, bt, 1.0), ValueError),
                        ((_t(2, 1, 51, 128), c, n, bt, 1.0), ValueError), ((_t(2, 1, 6, 64), c, n, bt, 1.0), ValueError),
                        ((_t(3, 1, 6, 128), c, n, bt, 1.0), ValueError), ((q.half(), c, n, bt, 1.0), TypeError),
                        ((q, c, _i(2, 2), bt, 1.0), ValueError), ((q, c, n.bool(), bt, 1.0), TypeError),
                        ((q, c, n, bt, 1.0, _t(2, 1, 6, 64)), ValueError)]:
            with pytest.raises(e):
                wgkv.paged_decode_kv4(*args)


def test_operators_propagate_shapes():
    with FakeTensorMode():
        c, bt, n = _t(9, 16, 80, dtype=torch.uint8), _i(2, 3, 4), _i(2, 3)
        k, q = _t(2, 3, 5, 64), _t(2, 1, 6, 64)
        assert torch.ops.wgkv.paged_decode_kv4(q, c, n, bt, 0.1).shape == q.shape
        assert torch.ops.wgkv.kv4_append(k, k, c, n, bt, None) is None
        a, b = torch.ops.wgkv.kv4_read(c, None, n, bt, 5)
        assert a.shape == b.shape == (2, 3, 5, 64) and a.dtype == torch.bfloat16
        with pytest.raises(RuntimeError):
            torch.ops.wgkv.paged_decode_kv4(q, _t(9, 16, 81, dtype=torch.uint8), n, bt, 0.1)
        with pytest.raises(RuntimeError):
            torch.ops.wgkv.kv4_append(k, _t(2, 3, 4, 64), c, n, bt, None)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_oracle_rule(group):
    rng = np.random.default_rng(group)
    x = K4.bf16(rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1))) + rng.standard_normal((50, 1)))
    x[0] = 1.5                      # a constant row: scale 0, values exact
    x[1, 3] = np.nan                # spoilt rows read back as NaN
    x[2, 127] = -np.inf
    x[3, :2] = 3.3e38, -3.3e38      # a range that overflows
    x[3] = K4.bf16(x[3])
    code, lo, sc = K4.quantise(x, group)
    assert code.min() >= 0 and code.max() <= 15
    y = K4.values(code, lo, sc)
    assert np.array_equal(y[0], x[0]) and np.isnan(y[1:4]).all() and np.isfinite(y[4:]).all()
    step = np.repeat(sc, group, -1)[4:]
    # half a step and the rounding offset; the last code also carries the scale's own rounding (15 * 2^-9)
    assert (np.abs(y - x)[4:] <= step * (0.5 + 2.0 ** -12 + 15 * 2.0 ** -9)).all()
    # v half way between two codes goes up
    t = np.zeros((1, 128))
    t[0, :4] = 0, 15, 2.5, 7.5
    t[0, group - 1] = 15
    assert K4.quantise(t, group)[0][0, :4].tolist() == [0, 15, 3, 8]


@needs_lib
def test_call_by_array_checks_its_operation():
    assert lib.wgkv_kv4_call(3, F) == EINVAL and lib.wgkv_kv4_call(0, None) == EINVAL
    # the slot counts of the packed formats are the entry points' argument counts
    from wgkv import kv4
    for fmt, name in ((kv4._APPEND_SLOTS, "wgkv_kv4_append"), (kv4._READ_SLOTS, "wgkv_kv4_read"),
                      (kv4._DECODE_SLOTS, "wgkv_paged_decode_kv4")):
        assert fmt.size == 8 * len(lib.decls[name][1])
    # argument checks are reached through it too
    assert lib.wgkv_kv4_call(kv4._DECODE, kv4._DECODE_SLOTS.pack(F, F, 8, 24, 64, F, F, 4, 4, 1, 8, 2, 128, 1.0, F, F,
                                                                 1 << 30, F, 0)) == EINVAL
    assert lib.wgkv_stream_capture_id(None) == 0


def _pool(**kw):
    from wgkv.pool import WgkvPool
    p = WgkvPool()
    p.layers, p.batch, p.kv_heads, p.head_dim, p.window, p.page = 2, 3, 4, 128, 64, 16
    p.max_blocks_per_head, p.max_tokens_per_head, p.total_blocks = 100, 1600, 10000
    for n in ("block_table", "global_lengths", "local_is_global", "next_free_block", "err", "ring_state", "kv4"):
        setattr(p, n, F)
    p.kv4_group = 64
    for n, x in kw.items():
        setattr(p, n, x)
    return p


@needs_lib
def test_pool_entry_points_refuse_what_a_4_bit_pool_cannot_do():
    import ctypes

    def promote(**kw):
        p = _pool(**kw)
        return lib.wgkv_promote(ctypes.addressof(p), 64, None)  # the position is refused last: nothing launches

    assert promote() == EINVAL  # window 64: slot 64 does not exist
    for bad in (dict(kv4_group=16), dict(head_dim=64, kv4_group=128), dict(page=8), dict(kv4=F + 8),
                dict(quest_min=F), dict(free_ids=F, free_count=F), dict(kv4=None)):
        p = _pool(**bad)
        assert lib.wgkv_promote(ctypes.addressof(p), 3, None) == EINVAL, bad
    p = _pool(quest_min=F, quest_max=F)
    assert lib.wgkv_quest_select(ctypes.addressof(p), 0, 10, F, 0, 16, 144, F, F, 100, F, 1 << 20, None) == EINVAL
    p = _pool(free_ids=F, free_count=F)
    assert lib.wgkv_snapkv_evict(ctypes.addressof(p), F, 32, 16, 0.1, 0.3, 5, F, 1 << 30, None) == EINVAL


def test_pool_refusals():
    from types import SimpleNamespace
    from wgkv.layers import _kv_group
    kw = dict(layers=1, batch=1, kv_heads=2, head_dim=128, window=64, max_total_tokens=4096, max_tokens_per_head=1024,
              device="cpu")
    with pytest.raises(NotImplementedError):
        wgkv.init_pool(SimpleNamespace(), page=16, quest=True, kv_group=64, **kw)
    with pytest.raises(NotImplementedError):
        wgkv.init_pool(SimpleNamespace(), page=16, snapkv_window=32, q_heads=4, kv_group=64, **kw)
    with pytest.raises(TypeError):
        wgkv.init_pool(SimpleNamespace(), page=16, dtype=torch.float16, kv_group=64, **kw)
    with pytest.raises(ValueError):
        wgkv.init_pool(SimpleNamespace(), page=8, kv_group=64, **kw)
    with pytest.raises(ValueError):
        wgkv.init_pool(SimpleNamespace(), page=16, kv_group=48, **kw)
    assert _kv_group(SimpleNamespace()) is None and _kv_group(SimpleNamespace(kv_cache_bits=16)) is None
    assert _kv_group(SimpleNamespace(kv_cache_bits=4)) == 64
    assert _kv_group(SimpleNamespace(kv_cache_bits=4, kv_cache_group=32)) == 32
    with pytest.raises(ValueError):
        _kv_group(SimpleNamespace(kv_cache_bits=8))


@needs_lib
def test_decode_counts_the_records_of_divided_heads():
    # more than 8 query heads on a KV head are worked on as two heads: half as many records fit
    assert _decode(B=1024, Hk=4, Hq=32, width=(1 << 16) - 1, stride=1 << 16, page=32, nbytes=0) == ENOSPC
    assert _decode(B=1024, Hk=4, Hq=36, width=(1 << 16) - 1, stride=1 << 16, page=32, nbytes=0) == EINVAL
    assert _decode(B=1024, Hk=4, Hq=36, width=(1 << 15) - 1, stride=1 << 16, page=32, nbytes=0) == ENOSPC


@needs_lib
def test_decode_workspace_holds_every_counter():
    from wgkv import kv4
    assert kv4._COUNTER_BYTES == 2 * 4096 * 4  # the most heads, twice for divided ones
    assert lib.wgkv_paged_decode_kv4_workspace_size(1, 1, 1, 64) > kv4._COUNTER_BYTES
