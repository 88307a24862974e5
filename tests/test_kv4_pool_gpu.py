"""The paged pool held in 4 bits (``config.kv_cache_bits = 4``) through the framework's own path: prefill
admission, ring append, gate, promotion, deferred rescoring, decode attention, captured steps, the decoder.

A bf16 pool goes through the same calls.  Masks come from the bf16 keys, so page tables, lengths and the
allocator must agree exactly, and every row the 4-bit pool holds must be the quantised row of the bf16
pool (promotion moves codes, it does not round again); attention is held to the bound derived in
``kv4_oracle.decode`` on what the pool holds."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from golden_cases import O
from gpu_util import to_bf16
from kv4_util import held
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wgkv():
    import wgkv as m
    return m


def layers_of(wgkv, Ly, Hk, G, D, T, W, total, per_head, defer, seed, inputs=("pre_k",), **kw):
    cfg = SimpleNamespace(num_hidden_layers=Ly, num_key_value_heads=Hk, num_attention_heads=Hk * G, head_dim=D,
                          block_size=T, max_total_tokens=total, max_tokens_per_head=per_head, local_window_size=W,
                          g_defer=defer, g_threshold=0.5, **kw)
    torch.manual_seed(seed)
    out = []
    for l in range(Ly):
        gp = wgkv.GatingPredictor(D, Hk, list(inputs), "gelu", 64 / D, 1e-3, False, True).cuda().bfloat16()
        with torch.no_grad():
            gp.conv2.bias.fill_(0.1)
        out.append(wgkv.attach(SimpleNamespace(layer_idx=l, head_dim=D, scaling=D ** -0.5, g_predictors=gp), cfg))
    return out


TABLES = ("block_table", "global_lengths", "local_is_global", "next_free_block", "cache_seqlens")


def same_tables(a, b):
    for name in TABLES:
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert (a.local_length, a.local_ptr) == (b.local_length, b.local_ptr)


def positions(c, l, T, W):
    """Lengths (B, Hk) and tables of layer l as decode sees them."""
    lens = (c.local_length + c.global_lengths[l]).cpu().numpy()
    return lens, c.block_table[l].cpu().numpy()


def check_rows(c4, cb, Ly, D, group, T, W):
    """Every row the 4-bit pool holds is the bf16 pool's row, quantised."""
    kb, vb = (t.float().cpu().numpy().astype(np.float64) for t in (cb.block_pool_k, cb.block_pool_v))
    for l in range(Ly):
        lens, tbl = positions(c4, l, T, W)
        hk, hv = held(c4.block_pool_kv4, tbl, lens, D, group, T)
        for b in range(lens.shape[0]):
            for h in range(lens.shape[1]):
                pos = np.arange(lens[b, h])
                row = tbl[b, h, pos // T].astype(np.int64) * T + pos % T
                for got, src in ((hk, kb), (hv, vb)):
                    for x, y in zip(got[b][h], K4.quantise(src[row], group)):
                        np.testing.assert_array_equal(x, y)


def check_attention(out, q, c4, l, D, group, T, W):
    lens, tbl = positions(c4, l, T, W)
    hk, hv = held(c4.block_pool_kv4, tbl, lens, D, group, T)
    want, tol = K4.decode(q.float().cpu().numpy().transpose(0, 2, 1, 3), hk, hv, lens, D ** -0.5)
    got = out.double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)


@pytest.mark.parametrize("B,Ly,Hk,G,D,group,L,W,T,steps,defer,inputs", [
    (1, 2, 2, 4, 128, 64, 300, 64, 16, 150, False, ("pre_k",)),
    (2, 2, 3, 2, 64, 32, 75, 64, 32, 90, False, ("pre_k", "post_k", "v")),
    (1, 2, 2, 8, 128, 128, 40, 64, 16, 100, True, ("pre_k",)),      # prompt shorter than the decode phase's ring
    (2, 1, 2, 1, 128, 32, 2, 64, 16, 90, False, ("pre_k",)),        # the shortest prompt, one query head per KV head
])
def test_pool_path(wgkv, B, Ly, Hk, G, D, group, L, W, T, steps, defer, inputs):
    Hq = Hk * G
    per_head = W + L + steps + T
    args = (wgkv, Ly, Hk, G, D, T, W, Ly * B * Hk * per_head + 64 * T, per_head, defer, B + L, inputs)
    a4, ab = layers_of(*args, kv_cache_bits=4, kv_cache_group=group), layers_of(*args)
    c4, cb = SimpleNamespace(), SimpleNamespace()
    rng = np.random.default_rng(L + D)
    for l in range(Ly):
        x = [to_bf16(O.randn_bf16(rng, (B, L, h, D))).transpose(1, 2) for h in (Hq, Hk, Hk, Hk)]
        o4, ob = (a[l].self_attn_forward_patch(a[l], 3, None, c, (B, L), x[0], x[3], x[1], x[2])[0]
                  for a, c in ((a4, c4), (ab, cb)))
        # prefill attention reads the bf16 keys either way (by index here, from the pool there)
        torch.testing.assert_close(o4.float(), ob.float(), atol=2e-2, rtol=1e-2)
    torch.cuda.synchronize()
    wgkv.check_errors()
    assert c4.block_pool_k is None and cb.block_pool_kv4 is None
    same_tables(c4, cb)
    check_rows(c4, cb, Ly, D, group, T, W)
    for s in range(steps):
        outs = []
        for l in range(Ly):
            x = [to_bf16(O.randn_bf16(rng, (B, h, 1, D))) for h in (Hq, Hk, Hk, Hk)]
            o4, ob = (a[l].self_attn_forward_patch(a[l], 3, None, c, (B, 1), x[0], x[3], x[1], x[2])[0]
                      for a, c in ((a4, c4), (ab, cb)))
            outs.append((o4, x[0]))
        torch.cuda.synchronize()
        wgkv.check_errors()
        same_tables(c4, cb)
        if s % 7 == 0 or s == steps - 1:
            for l, (o, q) in enumerate(outs):
                check_attention(o, q, c4, l, D, group, T, W)
    check_rows(c4, cb, Ly, D, group, T, W)
    assert int(c4.global_lengths.sum()) > 0


def test_deferred_gate_on_post_rope_keys_reads_the_ring_back(wgkv):
    """With post_k and v among its inputs the gate rescores the ring on the values that the 4-bit pool holds."""
    B, Hk, D, W, T, group = 2, 2, 64, 64, 16, 32
    layers = layers_of(wgkv, 1, Hk, 2, D, T, W, 4096, 512, True, 3, ("pre_k", "post_k", "v"), kv_cache_bits=4,
                       kv_cache_group=group)
    a, c = layers[0], SimpleNamespace()
    rng = np.random.default_rng(0)
    x = [to_bf16(O.randn_bf16(rng, (B, h, 50, D))) for h in (4, Hk, Hk, Hk)]
    a.self_attn_forward_patch(a, 3, None, c, (B, 50), x[0], x[3], x[1], x[2])
    for _ in range(14):  # the last one fills slot W - 1 and rescores
        x = [to_bf16(O.randn_bf16(rng, (B, h, 1, D))) for h in (4, Hk, Hk, Hk)]
        a.self_attn_forward_patch(a, 3, None, c, (B, 1), x[0], x[3], x[1], x[2])
    torch.cuda.synchronize()
    wgkv.check_errors()
    ring = np.full((B, Hk), W, np.int32)
    hk, hv = held(c.block_pool_kv4, c.block_table[0].cpu().numpy(), ring, D, group, T)
    k, v = (to_bf16(np.stack([[K4.values(*h) for h in b] for b in x]).astype(np.float32)) for x in (hk, hv))
    want = torch.empty(B, Hk, W, dtype=torch.uint8, device="cuda")
    a.g_predictors.admit(c.local_pre_key[0], k, v, 0.5, want)
    assert torch.equal(c.local_is_global[0], want) and 0 < int(want.sum()) < want.numel()


@pytest.mark.parametrize("defer", [False, True])
def test_captured_steps_equal_eager_ones(wgkv, defer):
    B, Ly, Hk, G, D, L, W, T, n = 1, 3, 2, 4, 128, 100, 64, 16, 80
    per_head = W + L + n + T
    layers = layers_of(wgkv, Ly, Hk, G, D, T, W, Ly * B * Hk * per_head + 64 * T, per_head, defer, 5, kv_cache_bits=4)
    rng = np.random.default_rng(1)
    ce, cg = SimpleNamespace(), SimpleNamespace()
    for l in range(Ly):
        x = [to_bf16(O.randn_bf16(rng, (B, h, L, D))) for h in (Hk * G, Hk, Hk, Hk)]
        for c in (ce, cg):
            layers[l].self_attn_forward_patch(layers[l], 3, None, c, (B, L), x[0], x[3], x[1], x[2])
    g = torch.Generator(device="cuda").manual_seed(1)
    steps = torch.randn(n, Ly, 4, B, Hk * G, 1, D, generator=g, device="cuda").to(torch.bfloat16)
    s_in = torch.empty_like(steps[0])
    s_out = torch.empty(Ly, B, 1, Hk * G, D, dtype=torch.bfloat16, device="cuda")
    e_out = torch.empty_like(s_out)

    def run_step(cache, x, out):
        for l in range(Ly):
            o, _, _ = layers[l].self_attn_forward_patch(layers[l], 3, None, cache, (B, 1), x[l, 0], x[l, 3, :, :Hk],
                                                        x[l, 1, :, :Hk], x[l, 2, :, :Hk])
            out[l].copy_(o.reshape(out[l].shape))
        return out

    dg = wgkv.DecodeGraph(cg, W, defer=defer)
    for s in range(n):
        run_step(ce, steps[s], e_out)
        s_in.copy_(steps[s])
        got = s_out if s == 0 and dg.capture(lambda: run_step(cg, s_in, s_out)) is not None else dg.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, e_out), f"step {s}"
    wgkv.check_errors()
    same_tables(cg, ce)
    for l in range(Ly):  # codes and pairs of every row held, byte for byte
        lens, tbl = positions(ce, l, T, W)
        for x, y in zip(*(held(c.block_pool_kv4, tbl, lens, D, 64, T) for c in (ce, cg))):
            for b in range(B):
                for h in range(Hk):
                    for p, q in zip(x[b][h], y[b][h]):
                        np.testing.assert_array_equal(p, q)


def test_fused_prologue_quantises_the_same_rows(wgkv):
    """``self_attn_decode_fused`` (norm + RoPE + gate + append in one launch) on both pools."""
    B, Hk, G, D, W, T, L = 2, 2, 2, 128, 64, 16, 80
    args = (wgkv, 1, Hk, G, D, T, W, 8192, 512, False, 9)
    a4, ab = layers_of(*args, kv_cache_bits=4, kv_cache_group=32)[0], layers_of(*args)[0]
    c4, cb = SimpleNamespace(), SimpleNamespace()
    rng = np.random.default_rng(7)
    x = [to_bf16(O.randn_bf16(rng, (B, h, L, D))) for h in (Hk * G, Hk, Hk, Hk)]
    for a, c in ((a4, c4), (ab, cb)):
        a.self_attn_forward_patch(a, 3, None, c, (B, L), x[0], x[3], x[1], x[2])
    t = torch.outer(torch.arange(200.0, device="cuda"), 1.0 / 10000 ** (torch.arange(0, D, 2, device="cuda") / D))
    cos, sin = (torch.cat((f, f), -1).to(torch.bfloat16) for f in (t.cos(), t.sin()))
    for s in range(45):
        qkv = to_bf16(O.randn_bf16(rng, (B, (Hk * G + 2 * Hk) * D)))
        pos = torch.tensor([L + s], device="cuda")
        for a, c in ((a4, c4), (ab, cb)):
            a.self_attn_decode_fused(a, c, qkv, Hk * G, pos, cos, sin)
        torch.cuda.synchronize()
        wgkv.check_errors()
        same_tables(c4, cb)
    check_rows(c4, cb, 1, D, 32, T, W)


@pytest.mark.parametrize("defer", [False, True])
def test_decoder_runs_on_a_4_bit_pool(wgkv, defer):
    from wgkv.model import DecoderShape, WgkvDecoder
    shape = DecoderShape("tiny", 256, 2, 8, 2, 64, 512, 1000, 10000.0, False, 1e-5)
    m = WgkvDecoder(shape, batch=2, window=64, max_tokens_per_head=400, g_defer=defer, max_positions=400, kv_bits=4,
                    kv_group=32)
    ids = torch.randint(0, 1000, (2, 150), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    runs = []
    for graph in (False, True):
        c = SimpleNamespace()
        m.prefill(ids, c)
        toks = [m.token.clone()]
        if graph:
            dg = m.decode_graph(c)
            toks.append(m.token.clone())
            for _ in range(40):
                dg.replay()
                toks.append(m.token.clone())
        else:
            for _ in range(41):
                m.decode_step(c)
                toks.append(m.token.clone())
        torch.cuda.synchronize()
        wgkv.check_errors()
        assert c.block_pool_kv4 is not None and torch.isfinite(m.logits).all()
        runs.append(torch.cat(toks, 1))
    assert torch.equal(*runs)


def test_pool_capacity_errors_write_nothing(wgkv):
    """A prompt that does not fit flags the pool's error and leaves its bytes as they were."""
    Hk, D, W, T = 2, 64, 64, 16
    layers = layers_of(wgkv, 1, Hk, 2, D, T, W, 2 * W + 3 * T, 4096, False, 11, kv_cache_bits=4)
    a, c = layers[0], SimpleNamespace()
    with torch.no_grad():
        a.g_predictors.conv2.bias.fill_(5.0)  # everything admitted
    rng = np.random.default_rng(0)
    x = [to_bf16(O.randn_bf16(rng, (1, h, 300, D))) for h in (4, Hk, Hk, Hk)]
    a.self_attn_forward_patch(a, 3, None, c, (1, 300), x[0], x[3], x[1], x[2])
    with pytest.raises(AssertionError, match="pool exhausted"):
        wgkv.check_errors()
    assert not c.block_pool_kv4.any()
