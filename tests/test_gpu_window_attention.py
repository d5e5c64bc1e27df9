"""Attention through a window with sinks, over 16-bit and 4-bit pools, against 64-bit arithmetic."""
import ctypes
import math

import pytest
import torch

from helpers import assert_bits_equal
from oracle import q4_ref

pytestmark = pytest.mark.gpu


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def filled(device, bits, lens, H, rep, D, window, sinks, seed=1, **kw):
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(max(max(lens), 1) + 40, num_kv_heads=H, n_rep=rep, kv_bits=bits, window=window, sinks=sinks, **kw)
    k, v = rows(seed, len(lens), H, max(max(lens), 1), D), rows(seed + 1, len(lens), H, max(max(lens), 1), D)
    c.append_ragged(k.to(device), v.to(device), lens)
    return c, k, v


def check(out, q, k, v, lens, bits, window, sinks, mask=None, kv_start=None, what=""):
    out = out.double().cpu()
    assert torch.isfinite(out).all(), what
    held = q4_ref.values64 if bits == 4 else (lambda x: x.double())
    for b, n in enumerate(lens):
        ok = q4_ref.readable(n, q.shape[2], window, sinks, 0 if kv_start is None else kv_start[b], causal=mask is None)
        m = None if mask is None else mask[b if mask.shape[0] > 1 else 0, 0].expand(q.shape[2], -1)[:, :n].float()
        ref, parts = q4_ref.attention64(q[b], held(k[b, :, :n]), held(v[b, :, :n]), ok, m)
        worst = float(((out[b] - ref).abs() / q4_ref.error_bound(ref, parts, bits)).max())
        print(f"[window] {what} sequence {b}: {worst:.3f} of the bound")
        assert worst <= 1.0, f"{what} sequence {b}: {worst:.2f} of the bound"


SHAPES = [
    # D, KV heads, replicas, query tokens, lengths
    (128, 2, 4, 1, [1, 40, 700, 64]),
    (64, 3, 1, 5, [5, 129, 400]),
    (96, 1, 8, 2, [2, 260]),
    (256, 2, 2, 1, [33, 300]),
    (128, 2, 4, 100, [100, 612]),
    (64, 1, 8, 40, [64, 333]),
    (256, 1, 1, 50, [50, 170]),
    (128, 8, 4, 200, [200, 1000]),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D, H, rep, S, lens", SHAPES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (33, 4), (64, 0), (100, 37), (5000, 4)])
def test_window(device, bits, D, H, rep, S, lens, window, sinks):
    c, k, v = filled(device, bits, lens, H, rep, D, window, sinks)
    q = rows(3, len(lens), H * rep, S, D)
    check(c.attend(q.to(device)), q, k, v, lens, bits, window, sinks, what=f"{bits} D={D} S={S} w={window}+{sinks}")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("split", [32, 96])
def test_split_over_workgroups(device, bits, split):
    lens, H, rep, D = [1500, 700, 3], 2, 4, 128
    c, k, v = filled(device, bits, lens, H, rep, D, 600, 70)
    c.partition_tokens = split
    for S in (1, 3, 33):
        q = rows(3 + S, len(lens), H * rep, S, D)
        check(c.attend(q.to(device)), q, k, v, lens, bits, 600, 70, what=f"{bits} split {split} S={S}")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("window", [20, 200])
def test_mask_and_padding(device, bits, window):
    """A mask tensor and a window: both apply; left padding moves the sinks."""
    lens, H, rep, D, S, L = [90, 90], 2, 2, 128, 90, 90
    c, k, v = filled(device, bits, lens, H, rep, D, window, 3)
    q = rows(3, 2, H * rep, S, D)
    t = torch.arange(L)
    low = torch.finfo(torch.bfloat16).min
    mask = torch.stack([torch.where((t[None] <= t[:, None]) & (t[None] >= p), 0.0, low)[None] for p in (0, 31)]).bfloat16()
    check(c.attend(q.to(device), mask.to(device)), q, k, v, lens, bits, window, 3, mask=mask, what=f"{bits} mask")
    inf = mask.float().masked_fill(mask < -1, -math.inf)
    check(c.attend(q.to(device), inf.to(device)), q, k, v, lens, bits, window, 3, mask=inf, what=f"{bits} -inf mask")
    start = [0, 40]
    out = c.attend(q.to(device), kv_start=torch.tensor(start, dtype=torch.int32, device=device))
    check(out, q, k, v, lens, bits, window, 3, kv_start=start, what=f"{bits} kv_start")
    assert bool((out[1, :, :40] == 0).all()), "rows before the first readable token"


@pytest.mark.parametrize("bits", [16, 4])
def test_empty_and_short_sequences(device, bits):
    lens, H, rep, D, S = [0, 1, 2, 50], 2, 2, 64, 3
    c, k, v = filled(device, bits, lens, H, rep, D, 8, 2)
    q = rows(3, 4, H * rep, S, D)
    out = c.attend(q.to(device))
    assert bool((out[0] == 0).all()) and bool((out[1, :, :2] == 0).all()) and bool((out[2, :, :1] == 0).all())
    check(out[1:], q[1:], k[1:], v[1:], lens[1:], bits, 8, 2, what=f"{bits} short")


@pytest.mark.parametrize("S", [1, 4, 80])
def test_what_is_not_read_may_hold_anything(device, S):
    """Infinities and NaN between the sinks and the window, and behind the sequence, reach no output."""
    lens, H, rep, D, window, sinks = [200, 171], 2, 4, 128, 24, 5
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(256, num_kv_heads=H, n_rep=rep, window=window, sinks=sinks)
    k, v = rows(1, 2, H, 200, D), rows(2, 2, H, 200, D)
    for b, n in enumerate(lens):
        read = q4_ref.readable(n, S, window, sinks).any(0)
        bad = torch.tensor([math.nan, math.inf, -math.inf]).repeat(n)[:n].bfloat16()[None, :, None]
        k[b, :, :n] = torch.where(read[None, :, None], k[b, :, :n], bad)
        v[b, :, :n] = torch.where(read[None, :, None], v[b, :, :n], bad)
    # the pool's slots behind the sequences: written with infinities, then rolled back
    c.append_ragged(torch.full_like(k, math.inf).to(device), torch.full_like(v, math.nan).to(device), [200, 200])
    c.truncate([200, 200])
    c.append_ragged(k.to(device), v.to(device), lens)
    q = rows(3, 2, H * rep, S, D)
    check(c.attend(q.to(device)), q, k, v, lens, 16, window, sinks, what=f"garbage S={S}")


@pytest.mark.parametrize("bits", [16, 4])
def test_a_window_of_everything_changes_nothing(device, bits):
    lens, H, rep, D = [300, 41], 2, 4, 128
    c, k, v = filled(device, bits, lens, H, rep, D, None, 0)
    q = rows(3, 2, H * rep, 2, D)
    plain = c.attend(q.to(device))
    c.set_window(1000, 4)
    check(plain, q, k, v, lens, bits, 0, 0, what="plain")
    out = c.attend(q.to(device))
    check(out, q, k, v, lens, bits, 0, 0, what="wide window")
    if bits == 4:
        assert_bits_equal(out, plain, "the same kernel over the same units")


@pytest.mark.parametrize("bits", [16, 4])
def test_decode_steps_with_appends_and_capture(device, bits):
    """Decode steps through a window: eagerly, and captured and replayed past the window's length."""
    from pace_mi355.llm import KVCacheManager, KVCacheType

    class Cfg:
        num_hidden_layers = 2
        num_attention_heads = 8
        num_key_value_heads = 2

    B, D, P, steps, window, sinks = 2, 64, 20, 40, 24, 2
    mgr = KVCacheManager(Cfg(), 96, KVCacheType.PAGED, kv_bits=bits, window=window, sinks=sinks)
    mgr[1].set_window(None)  # layers may differ
    ks, vs = [[] for _ in range(2)], [[] for _ in range(2)]

    def feed(layer, seed, T):
        k, v, q = rows(seed, B, 2, T, D), rows(seed + 1, B, 2, T, D), rows(seed + 2, B, 8, T, D)
        ks[layer].append(k)
        vs[layer].append(v)
        return k, v, q

    def verify(layer, q, out, what):
        k, v = torch.cat(ks[layer], 2), torch.cat(vs[layer], 2)
        w, s = (window, sinks) if layer == 0 else (0, 0)
        check(out, q, k, v, [k.shape[2]] * B, bits, w, s, what=what)

    for i, T in enumerate((P, 1, 1)):
        for layer in range(2):
            k, v, q = feed(layer, 1000 * layer + 10 * i, T)
            mgr[layer].update_cache(k.to(device), v.to(device), 2)
            verify(layer, q, mgr[layer].attend(q.to(device)), f"eager {i}")
    k, v, q = (torch.zeros(2, B, h, 1, D, dtype=torch.bfloat16, device=device) for h in (2, 2, 8))

    def step():
        out = []
        for layer in range(2):
            mgr[layer].update_cache(k[layer], v[layer], 2)
            out.append(mgr[layer].attend(q[layer]))
        return out

    graph = mgr.capture_decode(step, steps)
    for i in range(steps):
        fresh = [feed(layer, 1000 * layer + 100 + 10 * i, 1) for layer in range(2)]
        for layer in range(2):
            k[layer].copy_(fresh[layer][0])
            v[layer].copy_(fresh[layer][1])
            q[layer].copy_(fresh[layer][2])
        got = graph.replay()
        torch.cuda.synchronize()
        if i % 9 == 0 or i == steps - 1:
            for layer in range(2):
                verify(layer, fresh[layer][2], got[layer], f"replay {i} layer {layer}")


def test_rotary_embedding_with_a_window(device):
    """A window takes the rotation in launches of its own; setting one between an append and its attention keeps the append."""
    from pace_mi355.llm import PagedKVCache
    from pace_mi355.ops import RotaryEmbedding

    B, H, rep, D, L = 2, 2, 4, 128, 60
    rope = RotaryEmbedding(None, D, 256, 10000.0)
    k, v, q = rows(1, B, H, L + 2, D), rows(2, B, H, L + 2, D), rows(3, B, H * rep, L + 2, D)
    call = rope(q.to(device), torch.arange(L + 2, device=device)[None].expand(B, -1).contiguous())
    qr, kr = (x.cpu() for x in call(q.to(device), k.to(device)))
    at = lambda lo, hi: rope(q.to(device), torch.arange(lo, hi, device=device)[None].expand(B, -1).contiguous())
    c = PagedKVCache(96, num_kv_heads=H, n_rep=rep, window=16, sinks=2)
    part = lambda x, lo, hi: x[:, :, lo:hi].to(device)
    c.update_cache(part(k, 0, L), part(v, 0, L), 2, rope=at(0, L))
    check(c.attend(part(q, 0, L)), qr[:, :, :L], kr[:, :, :L], v[:, :, :L], [L] * B, 16, 16, 2, what="prompt")
    c.update_cache(part(k, L, L + 1), part(v, L, L + 1), 2, rope=at(L, L + 1))
    c.set_window(None)
    check(c.attend(part(q, L, L + 1)), qr[:, :, L:L + 1], kr[:, :, :L + 1], v[:, :, :L + 1], [L + 1] * B, 16, 0, 0, what="window taken off")
    c.update_cache(part(k, L + 1, L + 2), part(v, L + 1, L + 2), 2, rope=at(L + 1, L + 2))
    c.set_window(7, 1)
    check(c.attend(part(q, L + 1, L + 2)), qr[:, :, L + 1:], kr, v, [L + 2] * B, 16, 7, 1, what="window set")


def test_blocks_beyond_two_gigabytes(device):
    B, H, D = 1, 8, 128
    nb = (9 << 30) // (H * 2 * 16 * D * 2)
    c, k, v = filled(device, 16, [0], H, 2, D, 40, 4, num_blocks=nb)
    alloc = c.state.allocator
    alloc.free(alloc.allocate(alloc.num_free))  # the highest ids come first now
    k, v, q = rows(3, B, H, 70, D), rows(4, B, H, 70, D), rows(5, B, 2 * H, 2, D)
    c.append_ragged(k.to(device), v.to(device), [70])
    assert int(c.state.table[0, :5].min()) > nb - 6
    check(c.attend(q.to(device)), q, k, v, [70], 16, 40, 4, what="high blocks")


def test_refused_over_fp32(device):
    from pace_mi355.llm import PagedKVCache

    x = torch.zeros(1, 2, 4, 64, device=device)
    with pytest.raises(RuntimeError, match="window over an fp32 pool"):
        PagedKVCache(64, window=8).update_cache(x, x, 2)
    c = PagedKVCache(64)
    c.update_cache(x, x, 2)
    with pytest.raises(RuntimeError, match="window over an fp32 pool"):
        c.set_window(8)
