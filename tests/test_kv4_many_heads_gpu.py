"""Decode attention near the most heads a call takes: the line of all heads then fills much of a CTA's shared
memory, and fewer CTAs fit on an SM."""
import numpy as np
import pytest
import torch

from kv4_util import dev, dev_i, kv_rows
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group,G,B,Hk,longest", [
    (128, 64, 4, 512, 8, 150), (128, 32, 1, 4096, 1, 150), (64, 64, 3, 1365, 3, 150), (128, 32, 8, 512, 8, 150),
    (64, 32, 16, 1024, 4, 150), (128, 32, 16, 512, 8, 150), (128, 64, 11, 455, 9, 150), (128, 128, 4, 850, 4, 3000)])
def test_decode_most_heads(D, group, G, B, Hk, longest):
    """Heads share 200 pages, in an order of their own; one in ten holds nothing."""
    import wgkv
    rng = np.random.default_rng(D + group + G + B)
    T, pages = 16, 200
    lens = rng.integers(1, longest + 1, (B, Hk)).astype(np.int32)
    lens[rng.random((B, Hk)) < 0.1] = 0
    lens[-1, -1] = longest
    cache = wgkv.kv4_alloc(pages, T, D, group)
    k, v = kv_rows(rng, 1, 1, pages * T, D), kv_rows(rng, 1, 1, pages * T, D)
    wgkv.kv4_append(dev(k), dev(v), cache, dev_i([[0]]), dev_i(np.arange(pages).reshape(1, 1, -1)))
    tbl = rng.integers(0, pages, (B, Hk, -(-longest // T))).astype(np.int32)
    q = K4.bf16(rng.standard_normal((B, 1, Hk * G, D)))
    args = dev(q), cache, dev_i(lens), dev_i(tbl), D ** -0.5
    out = wgkv.paged_decode_kv4(*args)
    again = wgkv.paged_decode_kv4(*args)
    torch.cuda.synchronize()
    wgkv.check_errors()
    assert torch.equal(out, again)
    parts = K4.unpack(cache.cpu().numpy(), D, group)
    slots = (tbl[..., None].astype(np.int64) * T + np.arange(T)).reshape(B, Hk, -1)
    got = out.double().cpu().numpy()
    picked = np.concatenate([rng.permutation(B)[:150], [0, B - 1]])  # sequences, wherever in the line
    for b in picked:
        hk = [[tuple(p[slots[b, h, :lens[b, h]]] for p in parts[:3]) for h in range(Hk)]]
        hv = [[tuple(p[slots[b, h, :lens[b, h]]] for p in parts[3:]) for h in range(Hk)]]
        want, tol = K4.decode(q[b:b + 1], hk, hv, lens[b:b + 1], D ** -0.5)
        over = np.abs(got[b:b + 1] - want) - tol
        assert (over <= 0).all(), f"sequence {b}: {(over > 0).sum()} outside, worst by {over.max():.3g}"
    empty = np.repeat(lens == 0, G, 1)
    assert not got[:, 0][empty].any() and got[:, 0][~empty].any(-1).all()


@pytest.mark.parametrize("D,group,G,B,Hk,width,T", [(64, 64, 1, 512, 8, 511, 4096), (64, 32, 8, 1, 60, 34900, 4096)])
def test_decode_most_records(D, group, G, B, Hk, width, T):
    """Just under 2^29 records of 16 tokens, the most a call takes: whole heads of one page over and over, so
    that every head's result is that of the page alone.

    A lane adds the same few numbers once for every pair of records that its warp takes, so fp32 sums of n terms
    are off by up to n 2^-24 of the terms' sizes, in the numerator and in the denominator."""
    import wgkv
    rng = np.random.default_rng(B)
    records = B * Hk * width * T // 16
    assert 0.99 * 2 ** 29 < records < 2 ** 29
    cache = wgkv.kv4_alloc(1, T, D, group)
    k, v = K4.bf16(0.1 * rng.standard_normal((1, 1, T, D))), K4.bf16(rng.standard_normal((1, 1, T, D)) + 2.0)
    wgkv.kv4_append(dev(k), dev(v), cache, dev_i([[0]]), dev_i([[[0]]]))
    q1 = K4.bf16(rng.standard_normal((1, 1, G, D)))
    table = torch.zeros(B, Hk, width, dtype=torch.int32, device="cuda")
    lens = torch.full((B, Hk), width * T, dtype=torch.int32, device="cuda")
    q = dev(q1).expand(B, Hk, G, D).reshape(B, 1, Hk * G, D)
    out = wgkv.paged_decode_kv4(q, cache, lens, table, D ** -0.5)
    torch.cuda.synchronize()
    wgkv.check_errors()
    parts = K4.unpack(cache.cpu().numpy(), D, group)
    want, tol = K4.decode(q1, [[tuple(parts[:3])]], [[tuple(parts[3:])]], np.array([[T]]), D ** -0.5)
    pairs = width * T / 32 / 4  # of a head, over the fewest warps of a CTA
    p_v = K4.values(parts[3], np.abs(parts[4]), parts[5]).max()
    tol = tol + 2 * min(pairs, records / 2 / 148 / 6) * 2.0 ** -24 * p_v
    got = out.double().cpu().numpy().reshape(-1, G, D)
    assert (np.abs(got - want.reshape(1, G, D)) <= tol.reshape(1, G, D)).all(), np.abs(got - want.reshape(1, G, D)).max()
