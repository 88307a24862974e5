"""What holding a cache in 4 bits costs: decode attention over the same rows held in bf16 and in 4 bits."""
import numpy as np
import pytest
import torch

from kv4_util import COMBOS, dev, dev_i
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


def predicted(q, k, v, group, scale):
    """Relative 2-norm of the difference for independent rows: a code is off by a uniform error of one step
    (step / sqrt(12) rms).  V's errors add to the output as V itself does, and K's move the scores by
    scale |q| (K's rms error), which moves the weights by as much, relative.  The denominator is V's own size."""
    D = q.shape[-1]
    rms = [np.sqrt((K4.quantise(x, group)[2] ** 2).mean() / 12) for x in (k, v)]
    return np.sqrt((rms[1] / v.std()) ** 2 + scale ** 2 * (q ** 2).mean() * D * rms[0] ** 2)


@pytest.mark.parametrize("D,group", COMBOS)
def test_difference_from_a_bf16_cache(D, group):
    """Rows of independent normal values (no structure that would help): the difference is what the steps of the
    codes make it, give or take the sampling of 32 heads and second-order terms (15 %)."""
    import wgkv
    rng = np.random.default_rng(D + group)
    B, Hk, G, n, T, scale = 4, 8, 4, 2000, 16, D ** -0.5
    k, v = (K4.bf16(rng.standard_normal((B, Hk, n, D))) for _ in range(2))
    q = K4.bf16(rng.standard_normal((B, 1, Hk * G, D)))
    pages = n // T
    table = dev_i(np.arange(B * Hk * pages).reshape(B, Hk, pages))
    lens = dev_i(np.full((B, Hk), n))
    kc, vc = (dev(x.reshape(B * Hk * pages, T, D)) for x in (k, v))
    want = wgkv.paged_decode(dev(q), kc, vc, lens, table, scale)
    cache = wgkv.kv4_alloc(B * Hk * pages, T, D, group)
    wgkv.kv4_append(dev(k), dev(v), cache, torch.zeros_like(lens), table)
    got = wgkv.paged_decode_kv4(dev(q), cache, lens, table, scale)
    torch.cuda.synchronize()
    wgkv.check_errors()
    want, got = (t.double().cpu().numpy() for t in (want, got))
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    expected = predicted(q, k, v, group, scale)
    print(f"D {D}, groups of {group}: off by {off:.4f} (2-norm, relative), expected {expected:.4f}")
    assert 0.85 * expected <= off <= 1.15 * expected
