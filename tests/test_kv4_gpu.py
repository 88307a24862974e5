"""The 4-bit KV cache on the GPU against its restatement in 64 bits (oracle/kv4_oracle.py).

Codes and pairs are compared exactly with the rule, bytes that no row owns stay as they were, read values
are the bf16 rounding of scale * code + minimum, and the attention is held to the bound that
``kv4_oracle.decode`` derives for every output."""
import numpy as np
import pytest
import torch

from kv4_util import COMBOS, dev, dev_i, filled, held, kv_rows, tables
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wgkv():
    import wgkv as m
    return m


def same_rows(got, want):
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)


def values32(c, lo, sc):
    """scale * code + minimum rounded to fp32, then to bf16 (float64 array)."""
    return K4.bf16(K4.values(c, lo, sc).astype(np.float32))


# ------------------------------------------------------------------------------------------- writing
@pytest.mark.parametrize("D,group", COMBOS)
@pytest.mark.parametrize("T,L,ragged", [(16, 1, False), (32, 37, True), (48, 200, True), (64, 16, False)])
def test_append_follows_the_rule_and_touches_nothing_else(wgkv, D, group, T, L, ragged):
    rng = np.random.default_rng(D + group + T + L)
    B, Hk = 2, 3
    start = rng.integers(0, 70, (B, Hk)).astype(np.int32)
    counts = rng.integers(0, L + 1, (B, Hk)).astype(np.int32) if ragged else np.full((B, Hk), L, np.int32)
    tbl, n = tables(rng, start + counts, T)
    k, v = kv_rows(rng, B, Hk, L, D), kv_rows(rng, B, Hk, L, D)
    cache = wgkv.kv4_alloc(n, T, D, group)
    cache.fill_(0xA5)
    before = K4.unpack(cache.cpu().numpy(), D, group)
    # (B, L, Hk, D) projections seen as (B, Hk, L, D)
    kt, vt = (dev(x.transpose(0, 2, 1, 3)).transpose(1, 2) for x in (k, v))
    out = wgkv.kv4_append(kt, vt, cache, dev_i(start), dev_i(tbl), dev_i(counts) if ragged else None)
    assert out is cache
    torch.cuda.synchronize()
    wgkv.check_errors()
    after = K4.unpack(cache.cpu().numpy(), D, group)
    own = np.zeros(n * T, bool)
    for b in range(B):
        for h in range(Hk):
            c = int(counts[b, h])
            pos = start[b, h] + np.arange(c)
            slot = tbl[b, h, pos // T].astype(np.int64) * T + pos % T
            own[slot] = True
            same_rows([p[slot] for p in after[:3]], K4.quantise(k[b, h, :c], group))
            same_rows([p[slot] for p in after[3:]], K4.quantise(v[b, h, :c], group))
    for a, z in zip(after, before):
        np.testing.assert_array_equal(a[~own], z[~own])


@pytest.mark.parametrize("D,group", COMBOS)
def test_append_special_rows(wgkv, D, group):
    rng = np.random.default_rng(5)
    k = kv_rows(rng, 1, 1, 24, D)
    k[0, 0, 0] = 0.0
    k[0, 0, 1] = -7.25                      # constant: scale 0
    k[0, 0, 2, 5] = np.nan
    k[0, 0, 3, D - 1] = np.inf
    k[0, 0, 4, 0] = -np.inf
    k[0, 0, 5, :2] = 3.3e38, -3.3e38        # range overflows
    k[0, 0, 6] *= 2.0 ** -130               # steps below 2^-126
    k[0, 0, 7] *= 2.0 ** 100
    k[0, 0, 8, ::2] = -0.0
    k[0, 0, 9, : D // 2] = 0.0
    k[0, 0, 10] = np.linspace(0, 15, D)     # many values half way between codes
    k[0, 0, 11] = np.tile(np.arange(32) * 0.5, D // 32)
    k = K4.bf16(k)
    v = k[:, :, ::-1].copy()
    lens = np.array([[24]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16, rows=(k, v))
    for got, x in ((hk[0][0], k), (hv[0][0], v)):
        c, lo, sc = K4.quantise(x[0, 0], group)
        same_rows([got[0], got[2]], [c, sc])
        np.testing.assert_array_equal(got[1], lo)  # NaN == NaN, -0.0 == 0.0 here


def test_append_alignments_and_strides(wgkv):
    """Rows at 2-byte alignment, strides that are no multiple of 8, a broadcast head, a reversed batch."""
    rng = np.random.default_rng(9)
    D, group, T, L = 128, 32, 16, 19
    x = dev(kv_rows(rng, 1, 1, 1, 60000)).view(-1)
    views = [x[1:1 + 2 * 3 * L * D].view(2, 3, L, D),
             torch.as_strided(x, (2, 3, L, D), (3 * L * 131, L * 131, 131, 1), 3),
             torch.as_strided(x, (2, 3, L, D), (L * D, 0, D, 1), 0)]
    start = np.array([[0, 5, 16], [7, 15, 31]], np.int32)
    tbl, n = tables(rng, start + L, T)
    for k in views:
        v = torch.as_strided(k, k.shape, k.stride(), k.storage_offset() + 2)
        cache, want = wgkv.kv4_alloc(n, T, D, group), wgkv.kv4_alloc(n, T, D, group)
        wgkv.kv4_append(k, v, cache, dev_i(start), dev_i(tbl))
        wgkv.kv4_append(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format),
                        want, dev_i(start), dev_i(tbl))
        assert torch.equal(cache, want) and cache.any()


def test_append_drops_what_has_no_place(wgkv):
    """Positions before or past the table and page ids outside the cache: dropped, flagged, the rest written."""
    rng = np.random.default_rng(3)
    D, group, T, L = 64, 32, 16, 20
    k = dev(kv_rows(rng, 1, 3, L, D))
    tbl = dev_i([[[0, 1], [2, 99], [-3, 4]]])
    for start, bit in (([[0, 0, 0]], "page id out of range"), ([[13, 0, 0]], "max_tokens_per_head"),
                       ([[-4, 0, 0]], "max_tokens_per_head"), ([[2 ** 31 - 5, 0, 0]], "max_tokens_per_head")):
        cache = wgkv.kv4_alloc(5, T, D, group)
        wgkv.kv4_append(k, k, cache, dev_i(start), tbl)
        with pytest.raises(AssertionError, match=bit):
            wgkv.check_errors()
        wgkv.check_errors()  # reported once
        got = K4.unpack(cache.cpu().numpy(), D, group)
        c, lo, sc = K4.quantise(k[0].double().cpu().numpy(), group)
        np.testing.assert_array_equal(got[0][32:48], c[1, :16])      # head 1, page 2: written
        np.testing.assert_array_equal(got[0][64:68], c[2, 16:])      # head 2, page 4: written
        s = int(start[0][0])
        rows = [r for r in range(L) if 0 <= s + r < 32]
        np.testing.assert_array_equal(got[0][[s + r for r in rows]], c[0][rows])


def test_append_moves_on_its_own_stream_and_in_graphs(wgkv):
    rng = np.random.default_rng(21)
    D, group, T = 128, 64, 16
    k = dev(kv_rows(rng, 2, 2, 1, D))
    start, tbl = dev_i([[0, 3], [17, 30]]), dev_i(np.arange(8).reshape(2, 2, 2))
    want = wgkv.kv4_append(k, k, wgkv.kv4_alloc(8, T, D, group), start, tbl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache = wgkv.kv4_alloc(8, T, D, group)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        wgkv.kv4_append(k, k, cache, start, tbl)
    side.synchronize()
    assert torch.equal(cache, want)
    x = torch.zeros_like(k)
    g = torch.cuda.CUDAGraph()
    cache.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        wgkv.kv4_append(x, x, cache, start, tbl)
    x.copy_(k)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


# ------------------------------------------------------------------------------------------- reading
@pytest.mark.parametrize("D,group", COMBOS)
@pytest.mark.parametrize("T", [16, 48])
def test_read_gives_the_values_and_zeros_behind(wgkv, D, group, T):
    rng = np.random.default_rng(D * group + T)
    lens = np.array([[100, 0, 33], [1, 64, 257]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, T)
    for start, rows in ((None, 257), (np.array([[3, 0, 31], [0, 63, 200]], np.int32), 60), (None, 1)):
        s = start if start is not None else np.zeros_like(lens)
        counts = lens - s
        out = tuple(torch.full((2, 3, rows, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        got = wgkv.kv4_read(cache, dev_i(start) if start is not None else None, dev_i(counts), dev_i(tbl), rows, out)
        fresh = wgkv.kv4_read(cache, dev_i(s), dev_i(counts).long(), dev_i(tbl).long(), rows)
        torch.cuda.synchronize()
        wgkv.check_errors()
        for o, f, x in zip(got, fresh, (hk, hv)):
            assert torch.equal(o, f)
            o = o.double().cpu().numpy()
            for b in range(2):
                for h in range(3):
                    m = min(int(counts[b, h]), rows)
                    a = slice(int(s[b, h]), int(s[b, h]) + m)
                    np.testing.assert_array_equal(o[b, h, :m], values32(*(p[a] for p in x[b][h])))
                    assert not o[b, h, m:].any()


def test_read_out_of_range(wgkv):
    rng = np.random.default_rng(2)
    cache, tbl, hk, _ = filled(wgkv, rng, np.array([[40, 40]], np.int32), 64, 64, 16)
    bad = tbl.copy()
    bad[0, 1, 1] = cache.shape[0]
    k, v = wgkv.kv4_read(cache, dev_i([[30, -2]]), dev_i([[30, 30]]), dev_i(bad), 30)
    with pytest.raises(AssertionError, match="page id out of range"):
        wgkv.check_errors()
    got = k.double().cpu().numpy()
    np.testing.assert_array_equal(got[0, 0, :10], values32(*(p[30:40] for p in hk[0][0])))
    assert not got[0, 0, 18:].any()          # past the three pages of the table
    np.testing.assert_array_equal(got[0, 1, 2:18], values32(*(p[:16] for p in hk[0][1])))
    assert not got[0, 1, :2].any() and not got[0, 1, 18:].any()


def test_nan_rows_read_as_nan(wgkv):
    rng = np.random.default_rng(4)
    k = kv_rows(rng, 1, 1, 20, 128)
    v = kv_rows(rng, 1, 1, 20, 128)
    k[0, 0, 3, 77] = np.nan
    v[0, 0, 19, 0] = np.inf
    cache, tbl, _, _ = filled(wgkv, rng, np.array([[20]], np.int32), 128, 32, 16, rows=(k, v))
    a, b = wgkv.kv4_read(cache, None, dev_i([[20]]), dev_i(tbl), 20)
    assert torch.isnan(a).any(-1).flatten().nonzero().flatten().tolist() == [3] and torch.isnan(a[0, 0, 3]).all()
    assert torch.isnan(b).any(-1).flatten().nonzero().flatten().tolist() == [19] and torch.isnan(b[0, 0, 19]).all()


# ----------------------------------------------------------------------------------------- attention
def attend(wgkv, q, cache, lens, tbl, scale, **kw):
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i(lens), dev_i(tbl), scale, **kw)
    torch.cuda.synchronize()
    wgkv.check_errors()
    return out.double().cpu().numpy()


def within(got, want, tol):
    assert np.isfinite(got).all()
    over = np.abs(got - want) - tol
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} outside, worst by {over.max():.3g}"


@pytest.mark.parametrize("D,group", COMBOS)
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 8), (6, 2), (32, 8), (5, 1), (7, 1), (8, 1), (18, 2), (16, 1)])
@pytest.mark.parametrize("B,T,longest", [(1, 16, 130), (3, 48, 1000)])
def test_decode(wgkv, D, group, Hq, Hk, B, T, longest):
    rng = np.random.default_rng(D + group + 17 * Hq + Hk + B + T)
    lens = rng.integers(0, longest + 1, (B, Hk)).astype(np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, T, fill=0xFF)  # unused places hold NaN pairs
    q = K4.bf16(rng.standard_normal((B, 1, Hq, D)))
    got = attend(wgkv, q, cache, lens, tbl, D ** -0.5)
    within(got, *K4.decode(q, hk, hv, lens, D ** -0.5))


@pytest.mark.parametrize("D,group", COMBOS)
def test_decode_lengths_around_the_records(wgkv, D, group):
    rng = np.random.default_rng(group)
    lens = np.array([[0, 1, 2, 15, 16, 17, 31, 32], [33, 47, 48, 63, 64, 65, -5, 129]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16, fill=0xFF)
    q = K4.bf16(rng.standard_normal((2, 1, 32, D)))
    got = attend(wgkv, q, cache, lens, tbl, D ** -0.5)
    want, tol = K4.decode(q, hk, hv, lens, D ** -0.5)
    within(got, want, tol)
    assert not got.reshape(2, 8, 4, D)[lens <= 0].any()


@pytest.mark.parametrize("D,group,Hq,Hk,B,longest", [(128, 64, 32, 8, 2, 20000), (64, 32, 32, 8, 1, 40000),
                                                     (128, 32, 16, 1, 3, 30011), (128, 128, 8, 8, 40, 3000),
                                                     (64, 64, 12, 1, 1, 9001)])
def test_decode_split_over_the_length(wgkv, D, group, Hq, Hk, B, longest):
    """Heads cut over many CTAs, several heads in one CTA, and lengths far apart."""
    rng = np.random.default_rng(longest)
    lens = rng.integers(1, longest + 1, (B, Hk)).astype(np.int32)
    lens[0, 0] = longest
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16)
    q = K4.bf16(rng.standard_normal((B, 1, Hq, D)) * 2)
    got = attend(wgkv, q, cache, lens, tbl, D ** -0.5)
    within(got, *K4.decode(q, hk, hv, lens, D ** -0.5))


@pytest.mark.parametrize("D,group,Hq,Hk,B", [(64, 64, 16, 4, 50), (128, 32, 10, 2, 40), (64, 32, 20, 2, 30), (64, 64, 8, 8, 60),
                                             (64, 32, 48, 8, 40), (128, 128, 16, 1, 150)])
def test_decode_many_unequal_heads(wgkv, D, group, Hq, Hk, B):
    """Long heads between very short ones: a CTA's segment holds parts of several, and its warps run ahead of
    one another where they end."""
    rng = np.random.default_rng(17)
    lens = rng.choice([0, 1, 16, 33, 70, 900, 5000], (B, Hk), p=[.1, .15, .15, .2, .1, .2, .1]).astype(np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16)
    q = K4.bf16(rng.standard_normal((B, 1, Hq, D)))
    args = dev(q), cache, dev_i(lens), dev_i(tbl), D ** -0.5
    out = wgkv.paged_decode_kv4(*args)
    again = [wgkv.paged_decode_kv4(*args) for _ in range(20)]
    torch.cuda.synchronize()
    wgkv.check_errors()
    within(out.double().cpu().numpy(), *K4.decode(q, hk, hv, lens, D ** -0.5))
    assert all(torch.equal(o, out) for o in again)


@pytest.mark.parametrize("D,group,G", [(128, 64, 4), (64, 32, 8), (128, 128, 12)])
def test_decode_long_flat_softmax_keeps_its_precision(wgkv, D, group, G):
    """Millions of records over V's that cancel: the result is hundreds of times smaller than the sums of
    codes behind it, so rounding that is biased (an accumulation that truncates) shows.

    The bound, in the 2-norm: the output's rounding to bf16 is uniform over half steps of at most 2^-8,
    2^-8 / sqrt(3) = 2.26e-3; the weights' rounding to fp16, at most 2^-11 each and independent, leaves
    2^-11 / sqrt(3) times rms(scale * code) / rms(v) = 2.5 for normal V, 7e-4; together 2.4e-3."""
    rng = np.random.default_rng(D + G)
    B, Hk, n, T = 16, 4, 54000, 16
    one = np.array([[n]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, one, D, group, T,
                                rows=[K4.bf16(rng.standard_normal((1, 1, n, D))) for _ in range(2)])
    q = K4.bf16(rng.standard_normal((B, 1, Hk * G, D)) * 0.3)
    shared = dev_i(tbl).expand(B, Hk, -1)  # every head on the same pages: 64 heads of work, one of memory
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i(np.full((B, Hk), n)), shared, D ** -0.5)
    wgkv.check_errors()
    k, v = K4.values(*hk[0][0]), K4.values(*hv[0][0])
    x = q.reshape(-1, D) @ k.T * D ** -0.5
    p = np.exp(x - x.max(-1, keepdims=True))
    want = (p @ v / p.sum(-1, keepdims=True)).reshape(q.shape)
    err = np.linalg.norm(out.double().cpu().numpy() - want) / np.linalg.norm(want)
    assert err <= 2.4e-3, err


@pytest.mark.parametrize("D,group", COMBOS)
def test_decode_extreme_values(wgkv, D, group):
    """Queries and rows of very different sizes: tokens whose V is tiny but whose weight is 1 next to huge
    V of no weight, constant rows, queries at the ends of bf16's useful range, a scale of either sign."""
    rng = np.random.default_rng(D - group)
    lens = np.array([[70, 70, 70, 70]], np.int32)
    k, v = kv_rows(rng, 1, 4, 70, D), kv_rows(rng, 1, 4, 70, D)
    v *= np.exp2(rng.integers(-12, 13, (1, 4, 70, 1)))
    k[0, 1] *= 2.0 ** 20
    v[0, 2] = K4.bf16(rng.standard_normal((70, 1)) * 100)  # constant rows: scale 0
    v[0, 3, 5] *= 2.0 ** 12
    v[0, 3, 9:] *= 2.0 ** -10
    k, v = K4.bf16(k), K4.bf16(v)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 32, rows=(k, v))
    q = rng.standard_normal((1, 1, 8, D))
    q[0, 0, 2:4] *= 2.0 ** -22
    q[0, 0, 4] *= 2.0 ** -100
    q[0, 0, 5] = 0.0
    q[0, 0, 6, 1:] *= 2.0 ** -35
    q[0, 0, 7] *= 6.0
    q = K4.bf16(q)
    for scale in (D ** -0.5, -0.25, 0.0, 1.0):
        got = attend(wgkv, q, cache, lens, tbl, scale)
        within(got, *K4.decode(q, hk, hv, lens, scale))


def test_decode_spoilt_rows_stay_in_their_head(wgkv):
    """A NaN row of K or V makes its own head's outputs NaN and no other's; behind the length it is not seen."""
    rng = np.random.default_rng(8)
    D, group = 128, 64
    lens = np.array([[50, 50, 50, 50]], np.int32)
    k, v = kv_rows(rng, 1, 4, 60, D), kv_rows(rng, 1, 4, 60, D)
    k[0, 0, 49, 3] = np.nan
    v[0, 2, 0, 100] = np.inf
    k[0, 3, 50:] = np.nan
    v[0, 3, 50:] = np.nan
    full = np.full_like(lens, 60)
    cache, tbl, hk, hv = filled(wgkv, rng, full, D, group, 16, rows=(k, v))
    q = K4.bf16(rng.standard_normal((1, 1, 8, D)))
    got = attend(wgkv, q, cache, lens, tbl, D ** -0.5)
    assert np.isnan(got[0, 0, [0, 1, 4, 5]]).all()
    with np.errstate(all="ignore"):
        want, tol = K4.decode(q, hk, hv, lens, D ** -0.5)
    for h in (2, 3, 6, 7):
        within(got[0, 0, h], want[0, 0, h], tol[0, 0, h])


def test_decode_reports_what_it_cannot_read(wgkv):
    rng = np.random.default_rng(6)
    lens = np.array([[40, 33]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, 64, 32, 16)
    q = K4.bf16(rng.standard_normal((1, 1, 4, 64)))
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i([[40, 100]]), dev_i(tbl), 0.125)
    with pytest.raises(AssertionError, match="max_tokens_per_head"):
        wgkv.check_errors()
    want, tol = K4.decode(q, hk, hv, lens, 0.125)
    within(out.double().cpu().numpy()[:, :, :2], want[:, :, :2], tol[:, :, :2])
    bad = tbl.copy()
    bad[0, 1, 2] = -1
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i(lens), dev_i(bad), 0.125)
    with pytest.raises(AssertionError, match="page id out of range"):
        wgkv.check_errors()
    within(out.double().cpu().numpy()[:, :, :2], want[:, :, :2], tol[:, :, :2])


def test_decode_layouts_of_its_arguments(wgkv):
    """Wider table rows, 64-bit indices, a strided query, queries and outputs given, pages shared by heads."""
    rng = np.random.default_rng(12)
    D, group, T = 128, 32, 16
    lens = np.array([[100, 77], [3, 100]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, T)
    q = K4.bf16(rng.standard_normal((2, 1, 8, D)))
    want = wgkv.paged_decode_kv4(dev(q), cache, dev_i(lens), dev_i(tbl), 0.1)
    wide = dev_i(np.concatenate([tbl, np.full((2, 2, 5), 10 ** 6, np.int32)], -1))
    ln, tb = dev_i(lens), dev_i(tbl)
    two = torch.empty(2, 1, 16, D, dtype=torch.bfloat16, device="cuda")
    two[:, :, ::2] = dev(q)
    off = torch.empty(q.size + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape).copy_(dev(q))
    out = torch.full_like(want, float("nan"))
    for args in [(dev(q), wide, ln), (dev(q), wide[:, :, :tbl.shape[2]], ln), (dev(q), tb.long(), ln.long()),
                 (two[:, :, ::2], tb, ln), (off, tb, ln), (dev(q), tb.permute(2, 0, 1).contiguous().permute(1, 2, 0), ln)]:
        assert torch.equal(wgkv.paged_decode_kv4(args[0], cache, args[2], args[1], 0.1), want)
    assert wgkv.paged_decode_kv4(dev(q), cache, ln, tb, 0.1, out=out) is out and torch.equal(out, want)
    shared = tb[:1, :1].expand(2, 2, -1)
    got = wgkv.paged_decode_kv4(dev(q), cache, dev_i([[100, 9], [100, 50]]), shared, 0.1)
    kk, vv = [[hk[0][0]] * 2] * 2, [[hv[0][0]] * 2] * 2
    torch.cuda.synchronize()
    wgkv.check_errors()
    within(got.double().cpu().numpy(), *K4.decode(q, kk, vv, np.array([[100, 9], [100, 50]]), 0.1))
    with pytest.raises(ValueError, match="aligned"):
        wgkv.paged_decode_kv4(dev(q), cache, ln, tb, 0.1, out=off)


def test_decode_repeats_to_the_bit_and_counters_reset(wgkv):
    rng = np.random.default_rng(13)
    small = (np.array([[30000, 17000]], np.int32), 32, 128, 64)   # few counters, long partial results
    large = (rng.integers(1, 500, (20, 8)).astype(np.int32), 8, 64, 32)
    cases = []
    for lens, Hq, D, group in (small, large):
        cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16)
        q = dev(K4.bf16(rng.standard_normal((lens.shape[0], 1, Hq, D))))
        cases.append((q, cache, dev_i(lens), dev_i(tbl), D ** -0.5))
    first = [wgkv.paged_decode_kv4(*c).clone() for c in cases]
    for _ in range(5):
        for c, f in zip(cases, first):
            assert torch.equal(wgkv.paged_decode_kv4(*c), f)


def test_decode_graphs_and_streams(wgkv):
    """Two graphs captured on one stream and replayed at the same time on two, with eager calls on a third:
    each has scratch of its own."""
    rng = np.random.default_rng(14)
    lens = np.array([[50000, 3], [20000, 9000]], np.int32)
    cache, tbl, _, _ = filled(wgkv, rng, lens, 64, 64, 16)
    ln, tb = dev_i(lens), dev_i(tbl)
    qs = [dev(K4.bf16(rng.standard_normal((2, 1, 8, 64)))) for _ in range(3)]
    want = [wgkv.paged_decode_kv4(q, cache, ln, tb, 0.125) for q in qs]
    graphs = []
    torch.cuda.synchronize()
    for q in qs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = wgkv.paged_decode_kv4(q, cache, ln, tb, 0.125)
        graphs.append((g, o))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(30):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = wgkv.paged_decode_kv4(qs[2], cache, ln, tb, 0.125)
    torch.cuda.synchronize()
    for (_, o), w in zip(graphs, want):
        assert torch.equal(o, w)
    assert torch.equal(third, want[2])


def test_decode_from_two_threads(wgkv):
    """Calls of different sizes from two threads take turns in one stream's scratch."""
    import threading
    rng = np.random.default_rng(15)
    cases = []
    for lens, Hq, D in ((np.array([[9000, 5000]], np.int32), 8, 128),
                        (rng.integers(1, 900, (24, 8)).astype(np.int32), 8, 64)):
        cache, tbl, _, _ = filled(wgkv, rng, lens, D, 64, 16)
        args = (dev(K4.bf16(rng.standard_normal((lens.shape[0], 1, Hq, D)))), cache, dev_i(lens), dev_i(tbl), D ** -0.5)
        cases.append((args, wgkv.paged_decode_kv4(*args)))
    wrong = []

    def work(args, want):
        for _ in range(200):
            if not torch.equal(wgkv.paged_decode_kv4(*args), want):
                wrong.append(1)

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_integers_past_32_bits_stay_out_of_range(wgkv):
    rng = np.random.default_rng(16)
    lens = np.array([[40, 33]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, 64, 32, 16)
    before = cache.clone()
    row = dev(kv_rows(rng, 1, 2, 1, 64))
    far = torch.tensor([[2 ** 32, -2 ** 32 + 1]], device="cuda")
    wgkv.kv4_append(row, row, cache, far, dev_i(tbl))
    with pytest.raises(AssertionError, match="max_tokens_per_head"):
        wgkv.check_errors()
    assert torch.equal(cache, before)
    q = K4.bf16(rng.standard_normal((1, 1, 4, 64)))
    ln = torch.tensor([[40, 2 ** 32 + 5]], device="cuda")
    out = wgkv.paged_decode_kv4(dev(q), cache, ln, dev_i(tbl), 0.125)
    with pytest.raises(AssertionError, match="max_tokens_per_head"):
        wgkv.check_errors()
    want, tol = K4.decode(q, hk, hv, lens, 0.125)
    within(out.double().cpu().numpy()[:, :, :2], want[:, :, :2], tol[:, :, :2])
    bt = dev_i(tbl).long()
    bt[0, 1, 0] += 2 ** 32
    k, v = wgkv.kv4_read(cache, None, dev_i(lens), bt, 40)
    with pytest.raises(AssertionError, match="page id out of range"):
        wgkv.check_errors()
    assert (k[0, 1, :16] == 0).all() and (v[0, 1, :16] == 0).all()


# ------------------------------------------------------------------------------- as they are used together
@pytest.mark.parametrize("D,group,T", [(128, 64, 16), (64, 32, 32)])
def test_prompt_then_tokens(wgkv, D, group, T):
    """A prompt in two chunks, then decode steps that append a token and attend over everything; rows
    behind each head's length are left as they were."""
    rng = np.random.default_rng(D)
    B, Hk, G, steps = 2, 2, 4, 20
    first = rng.integers(0, 40, (B, Hk)).astype(np.int32)
    second = rng.integers(0, 60, (B, Hk)).astype(np.int32)
    tbl, n = tables(rng, first + second + steps, T)
    cache = wgkv.kv4_alloc(n, T, D, group)
    cache.fill_(0xFF)
    bt, lens = dev_i(tbl), torch.zeros(B, Hk, dtype=torch.int32, device="cuda")
    for c in (first, second):
        k, v = dev(kv_rows(rng, B, Hk, 60, D)), dev(kv_rows(rng, B, Hk, 60, D))
        torch.ops.wgkv.kv4_append(k, v, cache, lens, bt, dev_i(c))
        lens += dev_i(c)
    for _ in range(steps):
        k, v = dev(kv_rows(rng, B, Hk, 1, D)), dev(kv_rows(rng, B, Hk, 1, D))
        q = K4.bf16(rng.standard_normal((B, 1, Hk * G, D)))
        wgkv.kv4_append(k, v, cache, lens, bt)
        lens += 1
        out = wgkv.paged_decode_kv4(dev(q), cache, lens, bt, D ** -0.5)
        assert torch.equal(out, torch.ops.wgkv.paged_decode_kv4(dev(q), cache, lens, bt, D ** -0.5))
        host = lens.cpu().numpy()
        hk, hv = held(cache, tbl, host, D, group, T)
        within(out.double().cpu().numpy(), *K4.decode(q, hk, hv, host, D ** -0.5))
        back, _ = torch.ops.wgkv.kv4_read(cache, lens - 1, torch.ones_like(lens), bt, 1)
        want = K4.bf16(K4.values(*K4.quantise(k.double().cpu().numpy(), group)).astype(np.float32))
        np.testing.assert_array_equal(back.double().cpu().numpy(), want)
    wgkv.check_errors()
    code = K4.unpack(cache.cpu().numpy(), D, group)[0].reshape(n, T, D)
    for b in range(B):
        for h in range(Hk):
            used = int(host[b, h])
            if used % T:
                assert (code[tbl[b, h, used // T], used % T:] == 15).all()
