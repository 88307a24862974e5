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
