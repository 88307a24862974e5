"""Cases of the operators over a paged KV cache held in 4 bits.

Three operators and their run together:

* ``append``: K/V rows are quantised as they are written behind what each (sequence, KV head) holds
  already, and the rows written are read back;
* ``read``: the rows of every head are read back as bf16;
* ``decode``: one query token per sequence attends over each head's ragged pages;
* ``step``: a decode step of one layer, the new token appended and then attended with the rest.

A cache is ``(num_pages, page_size, row_bytes)`` uint8, ``row_bytes = D + 8 * D / group``: K and V of a
token, 4 bits a value, with a bf16 (minimum, scale) pair for each group of consecutive dimensions.  A page
is a run of 16-token records [K codes | K pairs | V codes | V pairs].
"""
import functools
import os
import sys

import numpy as np
import torch

own = False

C15 = float(np.float32(1.0 / 15.0))
UP = 0.5 + 2.0 ** -12  # rounding offset of the codes: ties go up, whatever the precision of the quotient
TINY = 2.0 ** -126


@functools.cache
def _wgkv():
    sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wg-kv_b200"))
    import wgkv
    return wgkv


# ---------------------------------------------------------------- cases
def _case(name, kind, B, Hq, Hk, D, group, page, dist, lo, hi, zero=0.0, rows=1, ragged=False, lens_seed=1):
    c = {"kind": kind, "B": B, "Hq": Hq, "Hk": Hk, "D": D, "group": group, "page": page, "dist": dist, "lo": lo,
         "hi": hi, "zero": zero, "rows": rows, "ragged": ragged, "lens_seed": lens_seed}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one sequence just past its prompt, one layer of an 8B-shaped model: latency counts
        _case("decode_b1_short", "decode", 1, 32, 8, 128, 64, 16, "uniform", 1000, 3000),
        # one sequence of a 1B-shaped model (head size 64) after a 32K prompt, ragged admission
        _case("decode_b1_d64_32k", "decode", 1, 32, 8, 64, 32, 16, "beta", 4096, 32000),
        # a serving batch of an 8B-shaped model at 128K of context, ragged admission
        _case("decode_b16_128k", "decode", 16, 32, 8, 128, 64, 16, "beta", 4096, 131072),
        # the same shape at the finest groups, smaller batch
        _case("decode_b4_g32_64k", "decode", 4, 32, 8, 128, 32, 16, "beta", 4096, 65536),
        # 64 short mixed sequences, coarsest groups, heads that hold nothing yet among them
        _case("decode_b64_mixed", "decode", 64, 32, 8, 128, 128, 32, "uniform", 1, 8191, zero=0.05),
        # all 16 query heads on one KV head, odd lengths, larger pages
        _case("decode_b8_mqa", "decode", 8, 16, 1, 128, 32, 64, "uniform", 501, 30011),
        # the ring of one layer read back whole (rescoring it with a deferred gate)
        _case("read_ring_b1", "read", 1, 32, 8, 64, 32, 16, "fixed", 4096, 4096),
        # whole heads read back: prefix reuse by a consumer of bf16 rows
        _case("read_b4_32k", "read", 4, 32, 8, 128, 64, 16, "uniform", 1, 32749, zero=0.05),
        # a decode step's token for each head of a batch
        _case("append_token_b16", "append", 16, 32, 8, 128, 64, 16, "uniform", 0, 2000),
        # a prompt chunk behind what is there, each head with its own number of rows
        _case("append_chunk_b2", "append", 2, 32, 8, 64, 32, 32, "uniform", 0, 1000, rows=509, ragged=True),
        # a whole 64K prompt of one sequence
        _case("append_prompt_64k", "append", 1, 32, 8, 128, 64, 16, "fixed", 0, 0, rows=65536),
        # append + attention of one layer's decode step, 32 sequences
        _case("step_b32", "step", 32, 32, 8, 128, 64, 16, "beta", 2048, 32000),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi] spread over its logarithm."""
    return min(hi, max(lo, int(round(np.exp(rng.uniform(np.log(max(lo, 0.7)), np.log(hi + 0.3)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "read", "append", "step"])
    D = rng.choice([64, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= D])
    page = rng.choice([16, 32, 48, 64])
    Hk = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    B = _log_int(rng, 1, 64)
    # bounds the padded size of the plain form and the cache: below the largest listed cases
    rows, ragged, lo = 1, False, 1
    if kind == "append":
        rows = _log_int(rng, 1, min(65536, 400_000 // (B * Hk)))
        ragged = rng.random() < 0.5
        lo, hi = 0, _log_int(rng, 1, 4000)
    else:
        hi = _log_int(rng, 1, min(131072, (2_000_000 if kind == "read" else 6_000_000) // (B * Hk)))
    dist = rng.choice(["uniform", "beta", "fixed"])
    if dist == "fixed":
        lo = hi
    zero = rng.choice([0.0, 0.0, 0.1])
    return _case(None, kind, B, Hk * G, Hk, D, group, page, dist, lo, hi, zero, rows, ragged, rng.randrange(1 << 30))


def _lengths(case):
    """(tokens held, rows appended) of each (sequence, KV head): a property of the case, not of the seed."""
    rng = np.random.default_rng(case["lens_seed"])
    n, lo, hi = case["B"] * case["Hk"], case["lo"], case["hi"]
    if case["dist"] == "beta":
        lens = lo + np.floor(rng.beta(2.0, 8.0, n) * (hi - lo)).astype(np.int64)
    else:
        lens = rng.integers(lo, hi + 1, n)
    lens[rng.random(n) < case["zero"]] = 0
    rows = np.full(n, case["rows"] if case["kind"] in ("append", "step") else 0, np.int64)
    if case["ragged"]:
        rows = rng.integers(0, case["rows"] + 1, n)
    return lens, rows


# ---------------------------------------------------------------- the format, in elementary torch operations
def _quantise(x, group):
    """(..., D) -> codes (..., D) int32, minimum and scale (..., D / group) bf16."""
    f = x.float().unflatten(-1, (-1, group))
    lo, hi = f.amin(-1), f.amax(-1)
    scale = ((hi - lo) * C15).to(torch.bfloat16).float()
    scale = torch.where(scale >= TINY, scale, torch.zeros_like(scale))
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    code = torch.floor(((f - lo[..., None]) * inv[..., None] + UP).clamp(max=15.5))
    bad = ~torch.isfinite(hi - lo).all(-1, keepdim=True)
    nan = torch.full_like(lo, float("nan"))
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return (code.flatten(-2).to(torch.int32), torch.where(bad, nan, lo).to(torch.bfloat16),
            torch.where(bad, nan, scale).to(torch.bfloat16))


def _pairs_bytes(lo, scale):
    """(..., NG) minimum and scale -> (..., 4 NG) uint8."""
    return torch.stack([lo, scale], -1).contiguous().view(torch.uint8).flatten(-2)


def _nibbles_bytes(code):
    """(..., 2 n) codes -> (..., n) bytes, the even one in the low half."""
    c = code.unflatten(-1, (-1, 2))
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)


def _row_bytes(k, v, group):
    """Quantised rows (N, D): K codes (N, D/2), K pairs (N, 4 NG), V codes (N, D/2), V pairs, each in the
    order in which the record lists a token's bytes."""
    D = k.shape[-1]
    kc, kl, ks = _quantise(k, group)
    vc, vl, vs = _quantise(v, group)
    kb = _nibbles_bytes(kc).view(-1, D // 32, 4, 4).transpose(1, 2).reshape(-1, D // 2)  # (j, t, 4 bytes) -> (t, j)
    vb = _nibbles_bytes(vc).view(-1, D // 32, 8, 2).transpose(1, 2).reshape(-1, D // 2)  # (j, g, 2 bytes) -> (g, j)
    return kb, _pairs_bytes(kl, ks), vb, _pairs_bytes(vl, vs)


def _row_offsets(D, group, device):
    """Byte offsets in a record of a token's K codes, K pairs, V codes and V pairs: (16, n) each."""
    NG = D // group
    r = torch.arange(16, device=device)[:, None]
    half, t4, odd = r // 8, (r % 8) // 2, r % 2
    kc = r * (D // 2) + torch.arange(D // 2, device=device)
    kp = 8 * D + r * 4 * NG + torch.arange(4 * NG, device=device)
    e = torch.arange(D // 2, device=device)
    g, j, byte = e // (D // 16), (e // 2) % (D // 32), e % 2
    vc = 8 * D + 64 * NG + half * 4 * D + (g * 4 + t4) * (D // 8) + j * 4 + odd * 2 + byte
    vp = 16 * D + 64 * NG + r * 4 * NG + torch.arange(4 * NG, device=device)
    return kc, kp, vc, vp


def _write_rows(cache, k, v, group, page, slot):
    """Rows (N, D) into the cache at token slots (N,) = page * page_size + offset."""
    D = k.shape[-1]
    rec = 16 * (D + 8 * (D // group))
    flat = cache.view(-1)
    base = (slot // 16) * rec
    for data, off in zip(_row_bytes(k, v, group), _row_offsets(D, group, k.device)):
        flat[base[:, None] + off[slot % 16]] = data


def _read_blocks(rec, D, group):
    """Records (..., rec bytes) -> K, V values (..., 16, D) fp32."""
    NG, J = D // group, D // 32

    def half_bytes(b):
        return torch.stack([b & 15, b >> 4], -1).flatten(-2)

    def pairs(b):
        p = b.contiguous().view(torch.bfloat16).unflatten(-1, (16, NG, 2)).float()
        return p[..., 0, None], p[..., 1, None]

    a, b, c = 8 * D, 8 * D + 64 * NG, 16 * D + 64 * NG
    kc = half_bytes(rec[..., :a].unflatten(-1, (16, 4, J, 4)))  # token, t, j, 8 codes
    vc = half_bytes(rec[..., b:c].unflatten(-1, (2, 8, 4, J, 2, 2)))  # half, g, t4, j, odd, 4 codes
    n = kc.dim() - 4
    lead = list(range(n))
    kc = kc.transpose(-3, -2).flatten(-3)
    vc = vc.permute(*lead, n, n + 2, n + 4, n + 3, n + 1, n + 5).flatten(-3).flatten(n, n + 2)
    kl, ks = pairs(rec[..., a:b])
    vl, vs = pairs(rec[..., c:])
    return ((kc.unflatten(-1, (NG, group)).float() * ks + kl).flatten(-2),
            (vc.unflatten(-1, (NG, group)).float() * vs + vl).flatten(-2))


def _gather(cache, table, page, D, group, first, n):
    """Values of records first .. first + n of every head: (B, Hk, 16 n, D) fp32 each."""
    rec = 16 * (D + 8 * (D // group))
    blk = torch.arange(first, first + n, device=cache.device)
    pg = table[:, :, (blk * 16 // page).clamp(max=table.shape[2] - 1)].long().clamp(min=0)
    k, v = _read_blocks(cache.view(-1, rec)[pg * (page // 16) + blk % (page // 16)], D, group)
    return k.flatten(2, 3), v.flatten(2, 3)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    B, Hq, Hk, D, page = (case[k] for k in ("B", "Hq", "Hk", "D", "page"))
    group = case["group"]
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens, rows = _lengths(case)
    need = (lens + rows + page - 1) // page
    width = max(1, int(need.max()))
    total = int(need.sum()) + 3
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    table = np.full((B * Hk, width), -1, np.int64)
    table[np.arange(width)[None, :] < need[:, None]] = np.arange(int(need.sum()))
    table = torch.from_numpy(table).to(dev)
    table = torch.where(table >= 0, perm[table.clamp(min=0)], torch.full_like(table, -1, dtype=torch.int32))

    # keys with channels of their own size and offset, values without
    amp = torch.exp(0.5 * torch.randn(D, generator=gen, device=dev))
    off = torch.randn(D, generator=gen, device=dev)

    def kv(*shape):
        k = torch.randn(*shape, D, generator=gen, device=dev) * amp + off
        v = torch.randn(*shape, D, generator=gen, device=dev)
        return k.to(torch.bfloat16), v.to(torch.bfloat16)

    cache = torch.zeros(total, page, D + 8 * (D // group), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 20) // page)
    for p0 in range(0, total, step) if case["kind"] != "append" else ():  # every page, whether used or not
        n = min(step, total - p0)
        k, v = kv(n * page)
        rec = 16 * (D + 8 * (D // group))
        out = cache[p0:p0 + n].view(-1, rec)
        parts = [x.view(-1, 16, x.shape[-1]) for x in _row_bytes(k, v, group)]
        for x, o in zip(parts, _row_offsets(D, group, dev)):
            out[:, o.flatten()] = x.flatten(1)
    s = {"case": case, "cache": cache, "table": table.view(B, Hk, width).contiguous(),
         "lens": torch.from_numpy(lens).to(dev, torch.int32).view(B, Hk),
         "rows": torch.from_numpy(rows).to(dev, torch.int32).view(B, Hk)}
    s["ends"] = s["lens"] + s["rows"]
    s["ends_max"] = int((lens + rows).max())
    if case["kind"] in ("append", "step"):
        # projections of (sequence, token, head, dim), handed over as (sequence, head, token, dim) views
        k, v = kv(B, case["rows"], Hk)
        s["k"], s["v"] = k.transpose(1, 2), v.transpose(1, 2)
    if case["kind"] in ("decode", "step"):
        s["q"] = torch.randn(B, 1, Hq, D, generator=gen, device=dev).to(torch.bfloat16)
        s["scale"] = D ** -0.5
    return s


# ---------------------------------------------------------------- one pass
def _plain_append(s):
    case = s["case"]
    L, page = case["rows"], case["page"]
    at = torch.arange(L, device=s["k"].device)
    keep = at < s["rows"][..., None]
    pos = (s["lens"][..., None] + at)[keep].long()
    pg = s["table"].gather(2, ((s["lens"][..., None] + at) // page).clamp(max=s["table"].shape[2] - 1).long())[keep]
    _write_rows(s["cache"], s["k"][keep], s["v"][keep], case["group"], page, pg.long() * page + pos % page)


def _plain_read(s, start, counts, n):
    """Rows start .. start + counts of every head, zero behind them: (B, Hk, n, D) bf16."""
    case = s["case"]
    D, page = case["D"], case["page"]
    rec = 16 * (D + 8 * (D // case["group"]))
    at = torch.arange(n, device=start.device)
    keep = at < counts[..., None]
    pos = torch.where(keep, start[..., None] + at, torch.zeros_like(at, dtype=torch.int32)).long()
    if start is s["zero"]:
        k, v = _gather(s["cache"], s["table"], page, D, case["group"], 0, -(-n // 16))
        k, v = k[:, :, :n], v[:, :, :n]
    else:  # the rows' records, and of each the row's place
        pg = s["table"].gather(2, pos // page).long().clamp(min=0)
        k, v = _read_blocks(s["cache"].view(-1, rec)[pg * (page // 16) + (pos % page) // 16], D, case["group"])
        place = (pos % 16)[..., None, None].expand(*pos.shape, 1, D)
        k, v = k.gather(3, place)[..., 0, :], v.gather(3, place)[..., 0, :]
    return [torch.where(keep[..., None], x, torch.zeros_like(x)).to(torch.bfloat16) for x in (k, v)]


def _plain_decode(s, lens, longest):
    case = s["case"]
    B, Hk, D = case["B"], case["Hk"], case["D"]
    k, v = _gather(s["cache"], s["table"], case["page"], D, case["group"], 0, max(1, -(-longest // 16)))
    q = s["q"].float().view(B, Hk, -1, D)
    keep = (torch.arange(k.shape[2], device=k.device) < lens[..., None])[:, :, None]
    x = (q @ k.transpose(2, 3)) * s["scale"]
    x = torch.where(keep, x, torch.full_like(x, float("-inf")))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    v = torch.where(keep.transpose(2, 3), v, torch.zeros_like(v))
    out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.to(torch.bfloat16).view(B, 1, -1, D)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        w = _wgkv()
        if kind == "decode":
            return w.paged_decode_kv4(s["q"], s["cache"], s["lens"], s["table"], s["scale"])
        if kind == "read":
            return w.kv4_read(s["cache"], None, s["lens"], s["table"], s["ends_max"])
        w.kv4_append(s["k"], s["v"], s["cache"], s["lens"], s["table"], s["rows"])
        if kind == "append":
            return w.kv4_read(s["cache"], s["lens"], s["rows"], s["table"], case["rows"])
        return w.paged_decode_kv4(s["q"], s["cache"], s["ends"], s["table"], s["scale"])
    s["zero"] = torch.zeros_like(s["lens"])
    if kind == "decode":
        return _plain_decode(s, s["lens"], s["ends_max"])
    if kind == "read":
        return _plain_read(s, s["zero"], s["lens"], s["ends_max"])
    _plain_append(s)
    if kind == "append":
        return _plain_read(s, s["lens"], s["rows"], case["rows"])
    return _plain_decode(s, s["ends"], s["ends_max"])


def work(case):
    lens, rows = _lengths(case)
    D, G = case["D"], case["Hq"] // case["Hk"]
    row = D + 8 * (D // case["group"])  # a token's K and V in the cache
    heads = case["B"] * case["Hk"]
    b = f = 0
    if case["kind"] in ("append", "step"):
        b += int(rows.sum()) * (4 * D + row)
        f += int(rows.sum()) * 2 * D * 8  # two comparisons, subtract, multiply, add, bound, round, pack
    if case["kind"] == "append":
        b += int(rows.sum()) * row + heads * case["rows"] * 4 * D
        f += int(rows.sum()) * 4 * D
    if case["kind"] == "read":
        b += int(lens.sum()) * row + heads * int(lens.max()) * 4 * D
        f += int(lens.sum()) * 4 * D
    if case["kind"] in ("decode", "step"):
        n = int((lens + rows).sum())
        b += n * row + int(((lens + rows + case["page"] - 1) // case["page"]).sum()) * 4 + 4 * case["B"] * case["Hq"] * D
        f += n * 4 * D * G
    return {"bytes": b + 8 * heads, "flops": f}


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_rows(s, b, h, first, n):
    """K and V (n, D) float64 that the cache holds for one head from position `first` on: code by code from
    the format's description (byte and half of every value, then scale * code + minimum)."""
    case = s["case"]
    D, page, group = case["D"], case["page"], case["group"]
    NG = D // group
    dev = s["cache"].device
    pos = torch.arange(first, first + n, device=dev)
    pg = s["table"][b, h, pos // page].long()
    base = (pg * page + pos % page) // 16 * (16 * (D + 8 * NG))
    r = (pos % 16)[:, None]
    d = torch.arange(D, device=dev)[None, :]
    flat = s["cache"].view(-1)
    k_at = r * (D // 2) + d % 32 // 8 * (D // 8) + d // 32 * 4 + d % 8 // 2
    v_at = (8 * D + 64 * NG + r // 8 * 4 * D + (d % 32 // 4 * 4 + r % 8 // 2) * (D // 8) + d // 32 * 4
            + r % 2 * 2 + d % 4 // 2)
    out = []
    for at, pair0 in ((k_at, 8 * D), (v_at, 16 * D + 64 * NG)):
        code = (flat[base[:, None] + at].to(torch.int64) >> (d % 2 * 4)) & 15
        p_at = base[:, None] + pair0 + (r * NG + torch.arange(NG, device=dev)) * 4
        word = sum(flat[p_at + i].to(torch.int64) << (8 * i) for i in range(4))
        pair = [((word >> sh & 0xffff) << 16).to(torch.int32).view(torch.float32).double() for sh in (0, 16)]
        out.append(code.double() * pair[1].repeat_interleave(group, 1) + pair[0].repeat_interleave(group, 1))
    return out


def _exact_quantised(x, group):
    """What rows (n, D) stand for once quantised, in 64 bits (finite rows)."""
    f = x.double().view(x.shape[0], -1, group)
    lo = f.min(-1, keepdim=True).values
    scale = ((f.max(-1, keepdim=True).values - lo) * C15).to(torch.bfloat16).double()
    code = torch.floor(torch.minimum((f - lo) / scale + UP, torch.full_like(f, 15.5)))
    return torch.where(scale >= TINY, scale * code + lo, lo.expand_as(f)).view(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    lens, rows = _lengths(case)
    B, Hk, Hq, D = case["B"], case["Hk"], case["Hq"], case["D"]
    G, dev, kind = Hq // Hk, s["cache"].device, case["kind"]
    n = case["rows"] if kind == "append" else int(lens.max())
    outs = ([torch.zeros(B, Hk, n, D, dtype=torch.float64, device=dev) for _ in range(2)]
            if kind in ("append", "read") else torch.zeros(B, 1, Hq, D, dtype=torch.float64, device=dev))
    for i in range(B * Hk):
        b, h = divmod(i, Hk)
        m, a = int(lens[i]), int(rows[i])
        new = [_exact_quantised(s[x][b, h, :a], case["group"]) for x in ("k", "v")] if a else []
        if kind == "append":
            for o, x in zip(outs, new):
                o[b, h, :a] = x
            continue
        old = _exact_rows(s, b, h, 0, m)
        if kind == "read":
            for o, x in zip(outs, old):
                o[b, h, :m] = x
            continue
        k, v = [torch.cat([x, y]) for x, y in zip(old, new)] if a else old
        if not len(k):
            continue
        p = torch.softmax((s["q"][b, 0, h * G:(h + 1) * G].double() @ k.T) * s["scale"], -1)
        outs[b, 0, h * G:(h + 1) * G] = p @ v
    return outs
