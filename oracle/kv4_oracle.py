"""Numpy restatement, in 64 bits, of the 4-bit KV cache: its rule of rounding, its record layout, and the
attention over it (include/wgkv.h, wgkv_kv4_*).  Test infrastructure only."""
from __future__ import annotations

import numpy as np

UP = 0.5 + 2.0 ** -12
C15 = float(np.float32(1.0 / 15.0))


def bf16(x):
    """Float64 values of x rounded to bf16 (nearest, ties to even; fp32 first is exact for what is passed here)."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.float32(np.nan), r).astype(np.float64)


def quantise(x, group):
    """Rows (..., D) -> (codes (..., D) int, minimum, scale (..., D / group) float64)."""
    x = np.asarray(x, np.float64)
    f = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        lo, hi = f.min(-1), f.max(-1)  # NaN where there is one
        rng = (hi.astype(np.float32) - lo.astype(np.float32)).astype(np.float64)
        scale = bf16((rng.astype(np.float32) * np.float32(C15)))
        scale = np.where(scale >= 2.0 ** -126, scale, 0.0)
        q = np.where(scale[..., None] > 0, (f - lo[..., None]) / np.where(scale > 0, scale, 1.0)[..., None], 0.0)
        code = np.floor(np.minimum(q + UP, 15.5))
    bad = ~np.isfinite(rng).all(-1)
    code[bad] = 0
    lo, scale = lo.copy(), scale.copy()
    lo[bad] = scale[bad] = np.nan
    return code.reshape(x.shape).astype(np.int64), lo, scale


def values(code, lo, scale):
    g = code.shape[-1] // lo.shape[-1]
    return code * np.repeat(scale, g, -1) + np.repeat(lo, g, -1)


def _bits(x):
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def unpack(cache, D, group):
    """Cache bytes (pages, page, row_bytes) -> K codes, min, scale, V codes, min, scale, token-major
    (pages * page, ...), value by value from the stated layout."""
    NG, W = D // group, D // 32
    rec = 16 * (D + 8 * NG)
    r = np.ascontiguousarray(cache).reshape(-1, rec)
    n = r.shape[0]
    out = []
    for which in (0, 1):
        code = np.zeros((n, 16, D), np.int64)
        for tok in range(16):
            for d in range(D):
                j, x = divmod(d, 32)
                if which == 0:
                    at, sh = tok * (D // 2) + (x // 8) * (D // 8) + 4 * j + (x % 8) // 2, 4 * (x % 2)
                else:
                    half, t4, odd = tok // 8, (tok % 8) // 2, tok % 2
                    at = 8 * D + 64 * NG + half * 4 * D + (4 * (x // 4) + t4) * (D // 8) + 4 * j + 2 * odd + (x % 4) // 2
                    sh = 4 * (x % 2)
                code[:, tok, d] = (r[:, at] >> sh) & 15
        p0 = 8 * D if which == 0 else 16 * D + 64 * NG
        pr = np.ascontiguousarray(r[:, p0:p0 + 64 * NG]).view(np.uint16).reshape(n, 16, NG, 2)
        f = (pr.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        out += [code.reshape(-1, D), f[..., 0].reshape(-1, NG), f[..., 1].reshape(-1, NG)]
    assert W * 32 == D
    return out


def decode(q, k, v, lens, scale):
    """Attention of q (B, 1, Hq, D) over k[b][h], v[b][h]: (codes, minimum, scale) of each head's tokens.
    Returns the output (B, 1, Hq, D) float64 and an error bound for a kernel that rounds the output to
    bf16 (half a step: 2^-8 relative), the weights p_t scale_t to fp16 (2^-11) and sums in fp32: a score is
    a sum of at most 2 D products, each rounding 2^-23 relative to the sum of the terms' sizes, times the
    few such sums it goes through (2^-20 in all), and enters the output twice (numerator, denominator)."""
    B, _, Hq, D = q.shape
    Hk = lens.shape[1]
    G = Hq // Hk
    out, tol = np.zeros(q.shape, np.float64), np.zeros(q.shape, np.float64)
    for b in range(B):
        for h in range(Hk):
            n = int(lens[b, h])
            if n <= 0:
                continue
            (kc, kl, ks), (vc, vl, vs) = k[b][h], v[b][h]
            kc, kl, ks, vc, vl, vs = (a[:n] for a in (kc, kl, ks, vc, vl, vs))
            sl = slice(h * G, (h + 1) * G)
            qq = q[b, 0, sl].astype(np.float64)
            x = qq @ values(kc, kl, ks).T * scale
            with np.errstate(invalid="ignore"):
                p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[b, 0, sl] = p @ values(vc, vl, vs)
            size_x = (np.abs(qq) @ values(kc, np.abs(kl), ks).T * abs(scale)).max(-1, keepdims=True)
            size_v = p @ values(vc, np.abs(vl), vs)
            tol[b, 0, sl] = 2.0 ** -8 * np.abs(out[b, 0, sl]) + (2.0 ** -11 + 2.0 ** -18 + 2 * 2.0 ** -20 * size_x) * size_v
    return out, tol
