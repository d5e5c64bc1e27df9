"""The 4-bit cache on the GPU: what is stored and read back bit for bit, attention over it against 64-bit arithmetic."""
import ctypes
import math

import numpy as np
import pytest
import torch

from helpers import assert_bits_equal
from oracle import q4_ref
from oracle.paged_ref import RaggedCacheModel

pytestmark = pytest.mark.gpu

SIZES = [64, 96, 128, 256]


def rows(seed, B, H, T, D, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, D, generator=g)
    if kind == "wide":
        x = x * torch.exp(2 * torch.randn(H, 1, D, generator=g))
    elif kind == "offset":
        x = 100 + 0.01 * x
    elif kind == "tiny":
        x = x * 2.0 ** -20
    elif kind == "equal":
        x = x[..., :1].expand(B, H, T, D).clone()
    elif kind == "ties":
        x = torch.randint(-30, 31, x.shape, generator=g) * 0.5  # quotients on the borders, over and over
    elif kind == "ends":
        x = x.bfloat16().float()
        pick = torch.randint(0, 40, x.shape, generator=g)
        for i, v in enumerate((math.inf, -math.inf, math.nan, 3.3e38, -3.3e38, 1e-38, -0.0, 32768.0)):
            x = torch.where(pick == i, torch.full_like(x, v), x)
    return x.bfloat16()


class Stored:
    """A 4-bit cache and the rows it should stand for."""

    def __init__(self, device, B, H, D, max_len, n_rep=1, **kw):
        from pace_mi355.llm import PagedKVCache

        self.device = device
        self.cache = PagedKVCache(max_len, num_kv_heads=H, n_rep=n_rep, kv_bits=4, **kw)
        self.model = RaggedCacheModel(B, H, D)  # rows as they were handed in
        self.n_rep = n_rep

    def append(self, k, v, counts=None, right=False):
        if counts is None:
            self.cache.update_cache(k.to(self.device), v.to(self.device), 2)
            self.model.append(k, v)
            return
        self.cache.append_ragged(k.to(self.device), v.to(self.device), counts, right_aligned=right)
        if right:
            T = k.shape[2]
            k, v = (torch.stack([torch.roll(x[b], -(T - c), dims=1) for b, c in enumerate(counts)]) for x in (k, v))
        self.model.append(k, v, counts)

    def expect(self, n_rep=1, pad_to=None):
        held = RaggedCacheModel(self.model.batch, *self.model.k[0].shape[::2])
        held.k = [q4_ref.values_bf16(x) for x in self.model.k]
        held.v = [q4_ref.values_bf16(x) for x in self.model.v]
        return held.dense(n_rep, pad_to)

    def check(self, what):
        k, v = self.cache.gather(n_rep=1)
        ek, ev = self.expect()
        assert_bits_equal(k, ek, what + " k")
        assert_bits_equal(v, ev, what + " v")

    def check_attention(self, q, out, what, mask=None, kv_start=None, window=0, sinks=0):
        out = out.double().cpu()
        assert torch.isfinite(out).all(), what
        for b in range(q.shape[0]):
            n = self.model.k[b].shape[1]
            start = 0 if kv_start is None else int(kv_start[b])
            ok = q4_ref.readable(n, q.shape[2], window, sinks, start, causal=mask is None)
            m = None if mask is None else mask[b if mask.shape[0] > 1 else 0, 0].expand(q.shape[2], -1)[:, :n].float()
            ref, parts = q4_ref.attention64(q[b], q4_ref.values64(self.model.k[b]), q4_ref.values64(self.model.v[b]), ok, m)
            err, bound = (out[b] - ref).abs(), q4_ref.error_bound(ref, parts, 4)
            worst = float((err / bound).max())
            print(f"[q4] {what} sequence {b}: {worst:.3f} of the bound")
            assert worst <= 1.0, f"{what}, sequence {b}: error {float(err.max()):.3e} is {worst:.2f} of its bound"


@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("kind", ["plain", "wide", "offset", "tiny", "equal", "ties", "ends"])
def test_rows_read_back_bit_for_bit(device, D, kind):
    B, H = 2, 3
    s = Stored(device, B, H, D, 128)
    for i, T in enumerate((5, 1, 2, 40, 1, 33)):  # half-filled blocks, single tokens, several blocks at once
        s.append(rows(10 * i, B, H, T, D, kind), rows(10 * i + 1, B, H, T, D, kind))
        s.check(f"{D} {kind} after {T}")


@pytest.mark.parametrize("D", SIZES)
def test_ragged_appends_by_slot(device, D):
    B, H = 4, 2
    s = Stored(device, B, H, D, 128)
    for i, counts in enumerate(([7, 0, 33, 1], [1, 1, 1, 1], [0, 20, 3, 15], [40, 40, 40, 40])):
        k, v = rows(100 + i, B, H, 40, D), rows(200 + i, B, H, 40, D, "wide")
        s.append(k, v, counts, right=i % 2 == 1)
        s.check(f"{D} step {i}")


def test_life_of_a_cache(device):
    """Rollback, eviction, compaction and forks move or forget stored rows like any other pool's."""
    B, H, D = 3, 2, 128
    s = Stored(device, B, H, D, 256)
    s.append(rows(1, B, H, 100, D), rows(2, B, H, 100, D))
    s.cache.truncate([3, 17, 50])
    s.model.truncate([3, 17, 50])
    s.check("rollback")
    s.append(rows(3, B, H, 9, D), rows(4, B, H, 9, D))
    s.check("append over rolled back rows")
    s.cache.evict_blocks(0, [1, 3])
    s.model.evict_blocks(0, [1, 3], 16)
    s.check("eviction")
    assert s.cache.compact() > 0
    s.check("compaction")
    for step in range(3):
        beams = [[1, 1, 0], [0, 0, 2], [2, 1, 0]][step]
        s.cache.reorder(beams)
        s.model.reorder(beams)
        s.append(rows(20 + step, B, H, 1, D), rows(30 + step, B, H, 1, D))
        s.check(f"fork {step}")


@pytest.mark.parametrize("D", [96, 128])
def test_gather_forms(device, D):
    B, H, lens = 4, 2, [0, 1, 37, 64]
    s = Stored(device, B, H, D, 80, n_rep=3)
    s.append(rows(1, B, H, 64, D), rows(2, B, H, 64, D), lens)
    ek, ev = s.expect(3, 70)
    k, v = s.cache.gather(pad_to=70)
    assert_bits_equal(k, ek, "dense")
    assert_bits_equal(v, ev, "dense v")
    pk, pv, cu = s.cache.gather_packed()
    assert cu.tolist() == [0, 0, 1, 38, 102]
    for b, n in enumerate(lens):
        assert_bits_equal(pk[cu[b]:cu[b + 1]], ek[b, :, :n].transpose(0, 1), f"packed {b}")
        assert_bits_equal(pv[cu[b]:cu[b + 1]], ev[b, :, :n].transpose(0, 1), f"packed v {b}")
    # rows behind a sequence keep what they held, and an out_len shorter than a sequence is not passed
    from pace_mi355 import _native as nat

    for out_len in (70, 20):
        ko = torch.full((B, H * 3, 70, D), 7.0, dtype=torch.bfloat16, device=device)
        vo = ko.clone()
        table, (lens_dev, bias) = s.cache.state.device_table(), s.cache.state.device_lens(s.cache.lens)
        nat.check(nat.load().pace_kv_gather_live(ctypes.byref(s.cache.pool_desc), table.data_ptr(), table.stride(0), lens_dev.data_ptr(), bias,
                                                 cu.data_ptr(), B, 3, ko.data_ptr(), vo.data_ptr(), ko.stride(0), ko.stride(1), out_len, 102,
                                                 nat.current_stream_ptr()))
        for b, n in enumerate(lens):
            m = min(n, out_len)
            assert_bits_equal(ko[b, :, :m], ek[b, :, :m], f"live {b}")
            assert_bits_equal(vo[b, :, :m], ev[b, :, :m], f"live v {b}")
            assert bool((ko[b, :, m:] == 7.0).all() and (vo[b, :, m:] == 7.0).all())


def test_strided_and_expanded_inputs(device):
    """[B, T, H, D] buffers seen as [B, H, T, D], and K/V expanded to the query heads."""
    B, H, T, D = 2, 2, 21, 64
    k, v = rows(1, B, H, T, D), rows(2, B, H, T, D)
    s = Stored(device, B, H, D, 64)
    kd, vd = (x.to(device).transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    s.cache.update_cache(kd, vd, 2)
    s.model.append(k, v)
    s.check("token-major")
    s2 = Stored(device, B, H, D, 64, n_rep=4)
    s2.cache.update_cache(k.repeat_interleave(4, 1).to(device), v.repeat_interleave(4, 1).to(device), 2)
    s2.model.append(k, v)
    s2.check("expanded")


CASES = [
    # D, KV heads, replicas, query tokens, lengths
    (128, 8, 4, 1, [1, 33, 500, 64]),
    (128, 2, 7, 1, [31, 1000]),
    (64, 3, 2, 5, [5, 6, 200]),
    (96, 4, 1, 1, [17, 90]),
    (256, 2, 1, 3, [3, 130, 300]),
    (128, 1, 16, 2, [40, 700]),
    (128, 2, 4, 40, [40, 41, 333]),
    (256, 1, 4, 33, [100, 64]),
    (64, 2, 8, 70, [70, 500]),
    (96, 1, 5, 64, [64, 129]),
    (128, 8, 4, 300, [300, 1100]),
]


@pytest.mark.parametrize("D, H, rep, S, lens", CASES)
@pytest.mark.parametrize("split", [0, 64])
def test_attention(device, D, H, rep, S, lens, split):
    B = len(lens)
    s = Stored(device, B, H, D, max(lens), n_rep=rep)
    s.append(rows(1, B, H, max(lens), D, "wide"), rows(2, B, H, max(lens), D), lens)
    s.cache.partition_tokens = split
    q = rows(3, B, H * rep, S, D)
    s.check_attention(q, s.cache.attend(q.to(device)), f"D={D} rep={rep} S={S} split={split}")


def test_the_new_token_is_read_as_it_is_stored(device):
    """A decode step: the append rides in the attention call and the token is attended to in its 4-bit form."""
    B, H, rep, D = 3, 2, 4, 128
    s = Stored(device, B, H, D, 128, n_rep=rep)
    s.append(rows(1, B, H, 30, D), rows(2, B, H, 30, D), [30, 0, 15])
    for step, T in enumerate((1, 1, 2, 32, 5)):
        k, v, q = rows(10 + step, B, H, T, D), rows(20 + step, B, H, T, D), rows(30 + step, B, H * rep, T, D)
        s.append(k, v)
        s.check_attention(q, s.cache.attend(q.to(device)), f"step {step}")
        s.check(f"step {step}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", [-math.inf, None])
def test_masks(device, dtype, low):
    """Additive masks with padding: rows masked everywhere are the average of what there is."""
    B, H, rep, D, S, L = 2, 2, 2, 128, 50, 50
    low = torch.finfo(dtype).min if low is None else low
    s = Stored(device, B, H, D, 64, n_rep=rep)
    s.append(rows(1, B, H, L, D), rows(2, B, H, L, D))
    q = rows(3, B, H * rep, S, D)
    t = torch.arange(L)
    mask = torch.zeros(B, 1, S, L, dtype=dtype)
    for b, pad in enumerate((0, 13)):
        mask[b, 0] = torch.where((t[None] <= t[:, None]) & (t[None] >= pad), 0.0, low)
    mask[0, 0, 20] = torch.randn(L)  # a bias that is not a padding mask
    s.check_attention(q, s.cache.attend(q.to(device), mask.to(device)), "padded mask", mask=mask)
    one = torch.randn(1, 1, 1, L).to(dtype)
    s.check_attention(q, s.cache.attend(q.to(device), one.to(device)), "broadcast mask", mask=one)


def test_kv_start_and_empty_rows(device):
    B, H, rep, D, S = 4, 2, 2, 64, 4
    lens = [0, 2, 60, 45]
    s = Stored(device, B, H, D, 64, n_rep=rep)
    s.append(rows(1, B, H, 60, D), rows(2, B, H, 60, D), lens)
    q = rows(3, B, H * rep, S, D)
    start = [0, 0, 58, 33]
    out = s.cache.attend(q.to(device), kv_start=torch.tensor(start, dtype=torch.int32, device=device))
    s.check_attention(q, out, "kv_start", kv_start=start)
    assert bool((out[0] == 0).all()), "a sequence without tokens"
    assert bool((out[1, :, :2] == 0).all()), "rows before the first token"
    assert bool((out[2, :, :2] == 0).all()), "rows before the first readable token"


@pytest.mark.parametrize("q_scale, kv_scale, kind", [(1e30, 1e-30, "plain"), (1e-30, 1.0, "plain"), (1e4, 1e-4, "plain"), (1.0, 1.0, "tiny"),
                                                     (64.0, 1.0, "offset")])
def test_ranges(device, q_scale, kv_scale, kind):
    """Queries and rows far from 1: a query row is brought into a half's range by itself."""
    B, H, D = 2, 2, 128
    s = Stored(device, B, H, D, 64)
    s.append((rows(1, B, H, 50, D, kind).float() * kv_scale).bfloat16(), rows(2, B, H, 50, D, kind))
    q = (rows(3, B, H, 1, D).float() * q_scale).bfloat16()
    s.check_attention(q, s.cache.attend(q.to(device)), f"{kind} {q_scale}")


def test_strided_queries_and_another_stream(device):
    B, H, rep, D, S, L = 2, 2, 4, 128, 3, 200
    s = Stored(device, B, H, D, 256, n_rep=rep)
    s.append(rows(1, B, H, L, D), rows(2, B, H, L, D))
    q = rows(3, B, H * rep, S, D)
    want = s.cache.attend(q.to(device))
    strided = q.to(device).transpose(1, 2).contiguous().transpose(1, 2)
    assert_bits_equal(s.cache.attend(strided), want, "token-major query")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = s.cache.attend(strided)
    torch.cuda.current_stream().wait_stream(side)
    assert_bits_equal(again, want, "side stream")
    s.check_attention(q, want, "strided")


def test_without_a_workspace(device):
    """Less scratch than asked for, or none: the context is cut over fewer workgroups."""
    from pace_mi355 import _native as nat

    B, H, rep, D, S, L = 1, 2, 4, 128, 2, 3000
    s = Stored(device, B, H, D, L, n_rep=rep)
    s.append(rows(1, B, H, L, D), rows(2, B, H, L, D))
    q = rows(3, B, H * rep, S, D)
    qd, lib = q.to(device), nat.load()
    table, lens_dev = s.cache.state.device_table(), torch.tensor([L], dtype=torch.int32, device=device)
    full = None
    for share in (1.0, 0.4, 0.0, "static"):
        out = torch.full_like(qd, math.nan)
        a = nat.PagedAttnArgs(q=qd.data_ptr(), q_stride_b=qd.stride(0), q_stride_h=qd.stride(1), q_stride_s=qd.stride(2), out=out.data_ptr(),
                              o_stride_b=out.stride(0), o_stride_h=out.stride(1), o_stride_s=out.stride(2), block_table=table.data_ptr(),
                              table_stride=table.stride(0), seq_lens=lens_dev.data_ptr(), batch=B, num_q_heads=H * rep, q_len=S, causal=1,
                              max_seq_len=L, scale=1 / math.sqrt(D))
        need = int(lib.pace_paged_attn_workspace_for(ctypes.byref(s.cache.pool_desc), ctypes.byref(a)))
        assert need > 0
        if share == "static":
            call = lib.pace_paged_attn_verify_static
        else:
            call = lib.pace_paged_attn_verify
            n = int(need * share)
            # a guard behind the part the library was told about
            ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = (ws.data_ptr(), n) if n else (None, 0)
        nat.check(call(ctypes.byref(s.cache.pool_desc), ctypes.byref(a), nat.current_stream_ptr()))
        if share != "static":
            assert bool((ws[n:] == 0x5A).all())
        s.check_attention(q, out, f"workspace {share}")


def test_blocks_beyond_two_gigabytes(device):
    """Offsets of a large pool do not fit 31 (or 32) bits."""
    B, H, D = 1, 8, 128
    nb = (5 << 30) // (H * 20 * D)
    s = Stored(device, B, H, D, 64, num_blocks=nb)
    s.append(rows(1, B, H, 1, D), rows(2, B, H, 1, D), [0])
    alloc = s.cache.state.allocator
    ids = alloc.allocate(alloc.num_free)
    alloc.free(ids)  # (a stack: the highest ids come first now)
    s.append(rows(3, B, H, 60, D), rows(4, B, H, 60, D))
    assert int(s.cache.state.table[0, :4].min()) > nb - 5
    s.check("high blocks")
    q = rows(5, B, H * 2, 2, D)
    s.n_rep = 2
    s.check_attention(q, s.cache.attend(q.to(device)), "high blocks")


def test_captured_decode_steps(device):
    """A decode step over 4-bit layers captured once and replayed, with the caller's own work between replays."""
    from pace_mi355.llm import KVCacheManager, KVCacheType

    class Cfg:
        num_hidden_layers = 2
        num_attention_heads = 8
        num_key_value_heads = 2

    B, D, P, steps = 2, 64, 20, 6
    eager, graphed = (KVCacheManager(Cfg(), 64, KVCacheType.PAGED, kv_bits=4) for _ in range(2))
    for layer in range(2):
        k, v, q = rows(layer, B, 2, P, D).to(device), rows(5 + layer, B, 2, P, D).to(device), rows(9, B, 8, P, D).to(device)
        for m in (eager, graphed):
            m[layer].update_cache(k, v, 2)
            m[layer].attend(q)
    k, v, q = (torch.zeros(2, B, h, 1, D, dtype=torch.bfloat16, device=device) for h in (2, 2, 8))

    def step(m):
        out = []
        for layer in range(2):
            m[layer].update_cache(k[layer], v[layer], 2)
            out.append(m[layer].attend(q[layer]))
        return out

    graph = graphed.capture_decode(lambda: step(graphed), steps)
    for i in range(steps):
        for x, h in ((k, 2), (v, 2), (q, 8)):
            x.copy_(torch.stack([rows(100 * i + layer + h, B, h, 1, D) for layer in range(2)]))
        want = step(eager)
        got = graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            # (the graph's partitions are sized for its last step: sums in another order, one step of bf16 at most)
            assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -9 * b.float().abs().amax()).all()), f"step {i}"
    for layer in range(2):
        for a, b in zip(graphed[layer].gather(), eager[layer].gather()):
            assert_bits_equal(a, b, "after replays")


def test_refused_uses(device):
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(64, kv_bits=4)
    x = torch.zeros(1, 2, 4, 64, device=device)
    with pytest.raises(RuntimeError, match="takes bf16"):
        c.update_cache(x, x, 2)
    c.update_cache(x.bfloat16(), x.bfloat16(), 2)
    with pytest.raises(RuntimeError, match="of the cache's dtype"):
        c.attend(x)
    with pytest.raises(RuntimeError, match="the cache holds"):
        c.update_cache(x, x, 2)


@pytest.mark.parametrize("D", [80, 128])
def test_a_model_run(device, D):
    """Prompt with padding mask, rotary embedding, decode, drafts, rollback, beams: the calls a model makes, through the
    attention operator, on a 4-bit cache."""
    from pace_mi355.llm import KVCacheManager, KVCacheType
    from pace_mi355.ops import MultiHeadAttention, RotaryEmbedding

    class Cfg:
        num_hidden_layers = 1
        num_attention_heads = 8
        num_key_value_heads = 2

    B, H, rep = 2, 2, 4
    pad = 96 if D == 80 else D  # rows are stored at a head size the kernels have, zeros behind the model's own
    mgr = KVCacheManager(Cfg(), 128, KVCacheType.PAGED, kv_bits=4)
    mha = MultiHeadAttention(dtype=torch.bfloat16)
    rope = RotaryEmbedding(None, D, 128, 10000.0)
    s = Stored(device, B, H, pad, 128, n_rep=rep)
    s.cache = mgr[0]
    widen = lambda x: torch.nn.functional.pad(x, (0, pad - x.shape[-1]))

    def step(seed, T, mask=None):
        at = len(mgr)
        k, v, q = rows(seed, B, H, T, D), rows(seed + 1, B, H, T, D), rows(seed + 2, B, H * rep, T, D)
        call = rope(v.to(device), torch.arange(at, at + T, device=device)[None].expand(B, T).contiguous())
        qr, kr = call(widen(q).to(device), widen(k).to(device))
        s.model.append(kr.cpu(), widen(v))
        pk, pv = mgr[0].update_cache(k.to(device), v.to(device), 2, rope=call)
        out = mha(q.to(device), pk, pv, mask)
        out = widen(out.cpu())
        # (1 / sqrt(D) of the model's head size: scale the wider rows' queries to match the oracle's)
        qq = qr.cpu().double() * math.sqrt(pad / D)
        for b in range(B):
            n = s.model.k[b].shape[1]
            ok = q4_ref.readable(n, T, causal=mask is None)
            m = None if mask is None else mask[b, 0, :, :n].float().cpu()
            ref, parts = q4_ref.attention64(qq[b], q4_ref.values64(s.model.k[b]), q4_ref.values64(s.model.v[b]), ok, m)
            ref[..., D:] = 0
            assert bool(((out[b].double() - ref).abs() <= q4_ref.error_bound(ref, parts, 4)).all()), f"seed {seed}"

    t = torch.arange(30)
    low = torch.finfo(torch.bfloat16).min
    mask = torch.stack([torch.where((t[None] <= t[:, None]) & (t[None] >= p), 0.0, low)[None] for p in (0, 11)]).bfloat16().to(device)
    step(1, 30, mask)
    for i in range(3):
        step(10 + 3 * i, 1)
    step(40, 5)
    mgr.remove_cache(3)
    s.model.truncate([3, 3])
    step(50, 1)
    mgr.update_cache_with_beam_indices(torch.tensor([1, 1]))
    s.model.reorder([1, 1])
    step(60, 1)
    step(70, 2)
