"""Decode attention over a 4-bit cache where V's scales and the probabilities are far apart at once: groups of
a row that differ by powers of two, a heavy token over a long flat tail."""
import numpy as np
import pytest
import torch

from kv4_util import dev, dev_i, filled
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


def spread_rows(rng, q, n, D, group, gap, nats, factor, scale):
    """K and V (1, 1, n, D) whose V groups behind the first are 2^-gap of it, with eight tokens whose scores are
    `nats` above the rest and whose first group is `factor` times as large."""
    k = rng.standard_normal((1, 1, n, D)) * 0.05
    v = rng.standard_normal((1, 1, n, D))
    v[..., group:] *= 2.0 ** -gap
    if nats:
        heavy = rng.permutation(n)[:8]
        k[0, 0, heavy] = q * nats / (scale * (q @ q))
        v[0, 0, heavy, :group] *= factor
    return K4.bf16(k), K4.bf16(v)


def range_tol(q, k, v, lens, scale):
    """What weights below fp16's normal numbers add to the bound of ``kv4_oracle.decode``: each is off by at most
    2^-25 in units in which the largest weight (probability times the token's largest scale) is at least
    2^6.5 (it is settled at 2^7, give or take a rounding of its exponent), for every code of the tokens."""
    B, _, Hq, D = q.shape
    Hk = lens.shape[1]
    G = Hq // Hk
    tol = np.zeros(q.shape)
    for b in range(B):
        for h in range(Hk):
            n = int(lens[b, h])
            kk, (vc, _, vs) = K4.values(*(a[:n] for a in k[b][h])), (a[:n] for a in v[b][h])
            x = q[b, 0, h * G:(h + 1) * G] @ kk.T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            top = (p * np.maximum(vs.max(-1), 2.0 ** -40)).max(-1, keepdims=True)
            tol[b, 0, h * G:(h + 1) * G] = top * 2.0 ** -31.5 * vc.sum(0)
    return tol


SPREADS = [(16, 0, 1), (20, 0, 1), (10, 8, 1), (12, 8, 1), (16, 8, 1), (8, 12, 1), (0, 12, 256), (12, 12, 1)]


@pytest.mark.parametrize("D,group,G", [(128, 64, 4), (128, 32, 8), (64, 32, 1)])
@pytest.mark.parametrize("gap,nats,factor", SPREADS)
def test_decode_scales_and_probabilities_far_apart(D, group, G, gap, nats, factor):
    import wgkv
    rng = np.random.default_rng(1000 * gap + 10 * nats + D + G)
    B, Hk, n, T, scale = 64, 4, 8000, 16, D ** -0.5
    base = rng.standard_normal(D)
    one = np.array([[n]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, one, D, group, T,
                                rows=spread_rows(rng, base, n, D, group, gap, nats, factor, scale))
    q1 = K4.bf16(base + 0.05 * rng.standard_normal((1, 1, G, D)))
    q = dev(q1).expand(B, Hk, G, D).reshape(B, 1, Hk * G, D)
    lens = dev_i(np.full((B, Hk), n))
    # every head on the same pages: a warp has thousands of tokens of one head before it
    out = wgkv.paged_decode_kv4(q, cache, lens, dev_i(tbl).expand(B, Hk, -1), scale)
    torch.cuda.synchronize()
    wgkv.check_errors()
    got = out.double().cpu().numpy().reshape(B * Hk, G, D)
    want, tol = K4.decode(q1, hk, hv, one, scale)
    tol = tol + range_tol(q1, hk, hv, one, scale)
    over = np.abs(got - want.reshape(1, G, D)) - tol.reshape(1, G, D)
    assert (over <= 0).all(), f"worst: {(np.abs(got - want.reshape(1, G, D)) / tol.reshape(1, G, D)).max():.3g} of the bound"


def one_token_rows(rng, n, D, G, size, sign):
    a = rng.integers(64, 120, n).astype(np.float64)
    a[rng.permutation(n)[0]] = 128 if sign > 0 else 48
    k = K4.bf16(a[:, None] * (1.0 + rng.integers(0, 8, D) / 8)).reshape(1, 1, n, D)
    return k, K4.bf16(rng.standard_normal((1, 1, n, D))), K4.bf16(np.full((1, 1, G, D), 2.0 ** (size - 14)))


@pytest.mark.parametrize("D,group,G,B,n", [(128, 64, 4, 1, 60), (128, 32, 8, 1, 60), (64, 64, 1, 1, 200),
                                           (128, 64, 4, 64, 2000), (64, 32, 8, 64, 2000), (128, 128, 12, 64, 2000)])
@pytest.mark.parametrize("size", [16, 22, 25, 28, 29, 30, 31, 32, 40])
@pytest.mark.parametrize("sign,v_size", [(1, 0), (-1, 0), (1, 6), (-1, -12)])
def test_decode_scores_of_any_size(D, group, G, B, n, size, sign, v_size):
    """Scores of about 2^size whose largest stands 2^-8 of that above the next: a softmax of one token, however
    coarse fp32 is at such scores (2^-24 of them; q k's products add up to a few of those).

    The result is that token's V, its codes' part through one weight that is rounded to fp16 (2^-11), the output
    rounded to bf16 (2^-8 of it at most), the rest in fp32."""
    import wgkv
    rng = np.random.default_rng(100 * size + D + G + n)
    T, Hk = 16, 4
    k, v, q1 = one_token_rows(rng, n, D, G, size, sign)
    one = np.array([[n]], np.int32)
    cache, tbl, hk, hv = filled(wgkv, rng, one, D, group, T, rows=(k, v * 2.0 ** v_size))
    x = q1[0, 0, 0] @ K4.values(*hk[0][0]).T * sign
    order = np.argsort(x)
    assert x[order[-1]] - x[order[-2]] > 2.0 ** -8 * np.abs(x).max() > 2.0 ** (size - 9)
    out = wgkv.paged_decode_kv4(dev(q1).expand(B, Hk, G, D).reshape(B, 1, Hk * G, D), cache,
                                dev_i(np.full((B, Hk), n)), dev_i(tbl).expand(B, Hk, -1), float(sign))
    wgkv.check_errors()
    got = out.double().cpu().numpy().reshape(-1, D)
    c, lo, sc = (t[order[-1]:order[-1] + 1] for t in hv[0][0])
    want, codes = K4.values(c, lo, sc), K4.values(c, 0 * lo, sc)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2.0 ** -18) * codes + 2.0 ** -20 * np.abs(want - codes)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
