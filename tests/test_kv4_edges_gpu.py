"""Calls of the 4-bit cache that its documentation allows: an output in the queries' place, the most heads of a
writer, queries that are not finite, calls on two forked streams of one graph."""
import numpy as np
import pytest
import torch

from kv4_util import dev, dev_i, filled, kv_rows
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wgkv():
    import wgkv as m
    return m


@pytest.mark.parametrize("D,group,Hq,Hk,B,longest", [(128, 64, 32, 8, 1, 3000), (64, 32, 8, 8, 40, 900),
                                                     (128, 32, 16, 1, 3, 9000), (64, 64, 1, 1, 1, 5)])
def test_decode_in_place_of_the_queries(wgkv, D, group, Hq, Hk, B, longest):
    rng = np.random.default_rng(D + Hq + B)
    lens = rng.integers(0, longest + 1, (B, Hk)).astype(np.int32)
    cache, tbl, _, _ = filled(wgkv, rng, lens, D, group, 16)
    q = dev(K4.bf16(rng.standard_normal((B, 1, Hq, D))))
    args = cache, dev_i(lens), dev_i(tbl), D ** -0.5
    want = wgkv.paged_decode_kv4(q, *args)
    for _ in range(5):
        x = q.clone()
        assert wgkv.paged_decode_kv4(x, *args, out=x) is x and torch.equal(x, want)
    wgkv.check_errors()


@pytest.mark.parametrize("D,group,Hq", [(128, 64, 8), (128, 32, 32), (64, 32, 12), (64, 64, 2)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_decode_spoilt_queries_stay_in_their_row(wgkv, D, group, Hq, value):
    """A query that is not finite spoils its own output and no other's (softmax of NaN or of infinity less
    infinity)."""
    rng = np.random.default_rng(D + Hq)
    lens = np.array([[3000, 70]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, lens, D, group, 16)
    q = K4.bf16(rng.standard_normal((1, 1, Hq, D)))
    want, tol = K4.decode(q, hk, hv, lens, D ** -0.5)
    bad = [1, Hq - 1]
    q[0, 0, bad] = value
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i(lens), dev_i(tbl), D ** -0.5)
    wgkv.check_errors()
    got = out.double().cpu().numpy()
    fine = [h for h in range(Hq) if h not in bad]
    assert np.isnan(got[0, 0, bad]).all()
    assert (np.abs(got - want) <= tol)[0, 0, fine].all()


def test_append_and_read_the_most_heads(wgkv):
    rng = np.random.default_rng(3)
    D, group, T, BH = 64, 64, 16, 65535
    k, v = (torch.randn(BH, 1, 1, D, device="cuda").bfloat16() for _ in range(2))
    start = torch.from_numpy(rng.integers(0, T, (BH, 1)).astype(np.int32)).cuda()
    table = torch.randperm(BH, device="cuda").to(torch.int32).view(BH, 1, 1)
    cache = wgkv.kv4_append(k, v, wgkv.kv4_alloc(BH, T, D, group), start, table)
    a, b = wgkv.kv4_read(cache, start, torch.ones_like(start), table, 1)
    wgkv.check_errors()
    for got, x in ((a, k), (b, v)):
        want = K4.bf16(K4.values(*K4.quantise(x.double().cpu().numpy(), group)).astype(np.float32))
        np.testing.assert_array_equal(got.double().cpu().numpy(), want)
    one = torch.zeros(65536, 1, dtype=torch.int32, device="cuda")
    rows = torch.zeros(65536, 1, 1, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="refused sizes"):
        wgkv.kv4_append(rows, rows, cache, one, one[:, :, None])
    with pytest.raises(ValueError, match="refused sizes"):
        wgkv.kv4_read(cache, None, one, one[:, :, None], 1)
    q = torch.zeros(4097, 1, 1, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="refused sizes"):
        wgkv.paged_decode_kv4(q, cache, one[:4097], one[:4097, :, None], 1.0)


def test_decode_on_forked_streams_of_one_graph(wgkv):
    """Two branches of a graph run at once, each with heads that are cut over many CTAs."""
    rng = np.random.default_rng(23)
    lens = np.array([[40000, 7], [30000, 9000]], np.int32)
    cache, tbl, _, _ = filled(wgkv, rng, lens, 64, 64, 16)
    ln, tb = dev_i(lens), dev_i(tbl)
    qs = [dev(K4.bf16(rng.standard_normal((2, 1, 8, 64)))) for _ in range(2)]
    want = [wgkv.paged_decode_kv4(q, cache, ln, tb, 0.125) for q in qs]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(3):
            got[0].append(wgkv.paged_decode_kv4(qs[0], cache, ln, tb, 0.125))
        with torch.cuda.stream(side):
            for _ in range(3):
                got[1].append(wgkv.paged_decode_kv4(qs[1], cache, ln, tb, 0.125))
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(20):
        g.replay()
    torch.cuda.synchronize()
    wgkv.check_errors()
    assert all(torch.equal(x, w) for xs, w in zip(got, want) for x in xs)
    assert all(torch.equal(wgkv.paged_decode_kv4(q, cache, ln, tb, 0.125), w) for q, w in zip(qs, want))


@pytest.mark.parametrize("D,group,G", [(128, 64, 4), (64, 64, 8)])
def test_decode_large_constant_values(wgkv, D, group, G):
    """Rows of V whose groups hold one value each (scale 0), up to the size that the documentation allows, next to
    scores that grow with every token so that the reference keeps moving: sums of p times V stay finite, and the
    output within the oracle's bound."""
    rng = np.random.default_rng(D)
    n = 1500
    one = np.array([[n]], np.int32)
    k = K4.bf16(0.1 * rng.standard_normal((1, 1, n, D)) + np.linspace(0, 2, n)[:, None])
    v = K4.bf16(np.repeat(2.0 ** 44 * rng.choice([-1.0, 1.0], (1, 1, n, D // group)), group, -1))
    cache, tbl, hk, hv = filled(wgkv, rng, one, D, group, 16, rows=(k, v))
    q = K4.bf16(1.0 + 0.1 * rng.standard_normal((1, 1, G, D)))
    out = wgkv.paged_decode_kv4(dev(q), cache, dev_i(one), dev_i(tbl), D ** -0.5)
    wgkv.check_errors()
    want, tol = K4.decode(q, hk, hv, one, D ** -0.5)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
