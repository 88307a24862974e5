"""Inputs of the 4-bit cache tests: ragged tables over permuted pages, rows at any alignment, and what the
oracle says a cache holds."""
import numpy as np
import torch

from oracle import kv4_oracle as K4

COMBOS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


def tables(rng, lens, T, spare=3):
    """A table (B, Hk, w) int32 giving every head its own permuted pages (-1 behind them), and the page count."""
    B, Hk = lens.shape
    need = (lens + T - 1) // T
    w = max(1, int(need.max()))
    n = int(need.sum()) + spare
    perm = rng.permutation(n).astype(np.int32)
    tbl = np.full((B, Hk, w), -1, np.int32)
    off = 0
    for b in range(B):
        for h in range(Hk):
            tbl[b, h, :need[b, h]] = perm[off:off + need[b, h]]
            off += need[b, h]
    return tbl, n


def kv_rows(rng, *shape):
    """bf16-exact float64 rows with channels of their own size and offset."""
    D = shape[-1]
    x = rng.standard_normal(shape) * np.exp(0.7 * rng.standard_normal(D)) + rng.standard_normal(D)
    return K4.bf16(x)


def dev(x, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


def dev_i(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def held(cache, tbl, lens, D, group, T):
    """What each head's pages hold by the stated layout: k[b][h], v[b][h] = (codes, minimum, scale)."""
    parts = K4.unpack(cache.cpu().numpy(), D, group)
    B, Hk = lens.shape
    k, v = [], []
    for b in range(B):
        k.append([])
        v.append([])
        for h in range(Hk):
            pos = np.arange(max(int(lens[b, h]), 0))
            slot = tbl[b, h, pos // T].astype(np.int64) * T + pos % T
            k[b].append(tuple(p[slot] for p in parts[:3]))
            v[b].append(tuple(p[slot] for p in parts[3:]))
    return k, v


def filled(wgkv, rng, lens, D, group, T, fill=None, rows=None):
    """A cache whose heads hold random rows of length lens: (cache, table (numpy), k, v as held)."""
    B, Hk = lens.shape
    tbl, n = tables(rng, np.maximum(lens, 0), T)
    cache = wgkv.kv4_alloc(n, T, D, group)
    if fill is not None:
        cache.fill_(fill)
    L = max(1, int(lens.max()))
    k, v = rows if rows is not None else (kv_rows(rng, B, Hk, L, D), kv_rows(rng, B, Hk, L, D))
    wgkv.kv4_append(dev(k), dev(v), cache, dev_i(np.zeros_like(lens)), dev_i(tbl), dev_i(lens))
    torch.cuda.synchronize()
    wgkv.check_errors()
    hk, hv = held(cache, tbl, lens, D, group, T)
    return cache, tbl, hk, hv
