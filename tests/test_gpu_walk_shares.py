"""How the attention kernels of the 4-bit cache and of the window deal a batch out to workgroups: batches of many and of empty
sequences, explicit cuts, workspaces of any size, several row groups, long single sequences, masks along a long context."""
import ctypes
import math

import pytest
import torch

from oracle import q4_ref

pytestmark = pytest.mark.gpu


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def filled(device, bits, lens, H, rep, D, window=None, sinks=0, seed=1):
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(max(max(lens), 1) + 40, num_kv_heads=H, n_rep=rep, kv_bits=bits, window=window, sinks=sinks)
    k, v = rows(seed, len(lens), H, max(max(lens), 1), D), rows(seed + 1, len(lens), H, max(max(lens), 1), D)
    c.append_ragged(k.to(device), v.to(device), lens)
    return c, k, v


def check(out, q, k, v, lens, bits, window=0, sinks=0, mask=None, what=""):
    out = out.double().cpu()
    assert torch.isfinite(out).all(), what
    held = q4_ref.values64 if bits == 4 else (lambda x: x.double())
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((out[b] == 0).all()), f"{what}: an empty sequence is zeros"
            continue
        ok = q4_ref.readable(n, q.shape[2], window, sinks, causal=mask is None)
        m = None if mask is None else mask[b if mask.shape[0] > 1 else 0, 0].expand(q.shape[2], -1)[:, :n].float()
        ref, parts = q4_ref.attention64(q[b], held(k[b, :, :n]), held(v[b, :, :n]), ok, m)
        worst = float(((out[b] - ref).abs() / q4_ref.error_bound(ref, parts, bits)).max())
        assert worst <= 1.0, f"{what} sequence {b} of {n}: {worst:.2f} of the bound"


@pytest.mark.parametrize("bits, window", [(4, None), (16, 300)])
@pytest.mark.parametrize("S", [1, 20])
@pytest.mark.parametrize("split", [0, 32, 160])
def test_many_sequences_some_empty(device, bits, window, S, split):
    """More groups than a wave has lanes, empty sequences at the ends, in the middle and in runs."""
    g = torch.Generator().manual_seed(3)
    lens = [0 if i in (0, 1, 63, 64, 65, 130, 149) else int(torch.randint(1, 400, (1,), generator=g)) for i in range(150)]
    c, k, v = filled(device, bits, lens, 1, 2, 64, window)
    c.partition_tokens = split
    q = rows(9, 150, 2, S, 64)
    check(c.attend(q.to(device)), q, k, v, lens, bits, window or 0, what=f"bits {bits} S={S} split {split}")


def test_all_empty(device):
    c, k, v = filled(device, 4, [0, 0, 0], 2, 2, 64)
    for split in (0, 32):
        c.partition_tokens = split
        for S in (1, 40):
            assert bool((c.attend(rows(1, 3, 4, S, 64).to(device)) == 0).all())


@pytest.mark.parametrize("bits, D", [(4, 128), (4, 256), (16, 64), (4, 96)])
@pytest.mark.parametrize("S", [1, 9, 130])
def test_one_long_sequence_among_short_ones(device, bits, D, S):
    lens = [6000, max(S, 7), 200, S]
    c, k, v = filled(device, bits, lens, 2, 4, D, None if bits == 4 else 5500)
    q = rows(9, 4, 8, S, D)
    check(c.attend(q.to(device)), q, k, v, lens, bits, 0 if bits == 4 else 5500, what=f"{bits} D={D} S={S}")


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("S, D", [(1, 128), (33, 128), (1, 256), (150, 64)])
def test_mask_along_a_long_context(device, bits, S, D):
    """Units that a mask leaves out in whole, at the front, in the middle and at the end; rows that it leaves nothing."""
    L, H, rep = 1400, 2, 2
    lens = [L, L]
    c, k, v = filled(device, bits, lens, H, rep, D, None if bits == 4 else L)
    low = torch.finfo(torch.bfloat16).min
    mask = torch.zeros(2, 1, S, L)
    mask[0, 0, :, :500] = low
    mask[0, 0, :, 700:900] = low
    mask[1, 0, :, 64:] = low
    mask[1, 0, S // 2, :] = low  # this row is the average of everything
    mask[0, 0, 0, 1390:] = torch.randn(10)
    q = rows(9, 2, H * rep, S, D)
    for m in (mask, mask.bfloat16()):
        check(c.attend(q.to(device), m.to(device)), q, k, v, lens, bits, 0 if bits == 4 else L, mask=m, what=f"{bits} S={S} {m.dtype}")


@pytest.mark.parametrize("S", [1, 9, 70])
def test_workspaces_of_any_size(device, S):
    """The library uses what it is given and nothing behind it, and the result does not depend on it beyond rounding."""
    from pace_mi355 import _native as nat

    lens, H, rep, D = [3000, 100, 0, 1700], 2, 4, 64
    c, k, v = filled(device, 4, lens, H, rep, D)
    q = rows(9, 4, H * rep, S, D)
    qd, lib = q.to(device), nat.load()
    table, lens_dev = c.state.device_table(), torch.tensor(lens, dtype=torch.int32, device=device)
    a = nat.PagedAttnArgs(q=qd.data_ptr(), q_stride_b=qd.stride(0), q_stride_h=qd.stride(1), q_stride_s=qd.stride(2), block_table=table.data_ptr(),
                          table_stride=table.stride(0), seq_lens=lens_dev.data_ptr(), batch=4, num_q_heads=H * rep, q_len=S, causal=1,
                          max_seq_len=3000, partition_tokens=256, scale=1 / math.sqrt(D))  # (cut whether that pays or not)
    need = int(lib.pace_paged_attn_workspace_for(ctypes.byref(c.pool_desc), ctypes.byref(a)))
    assert need > 0
    for size in (0, 1000, need // 50, need // 7, need // 2, need - 1, need, need + 4096):
        out = torch.full_like(qd, math.nan)
        ws = torch.full((size + 512,), 0x5A, dtype=torch.uint8, device=device)
        a.out, a.o_stride_b, a.o_stride_h, a.o_stride_s = out.data_ptr(), out.stride(0), out.stride(1), out.stride(2)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
        nat.check(lib.pace_paged_attn_verify(ctypes.byref(c.pool_desc), ctypes.byref(a), nat.current_stream_ptr()))
        assert bool((ws[size:] == 0x5A).all()), f"written behind a workspace of {size} bytes"
        check(out, q, k, v, lens, 4, what=f"S={S} workspace {size}")


def test_two_streams_with_workspaces_of_their_own(device):
    """Two calls that run side by side on different streams do not disturb each other."""
    from pace_mi355 import _native as nat

    lens, H, rep, D = [2500, 900], 2, 4, 128
    c, k, v = filled(device, 4, lens, H, rep, D)
    q = [rows(20 + i, 2, H * rep, 1, D) for i in range(2)]
    lib, table, lens_dev = nat.load(), c.state.device_table(), torch.tensor(lens, dtype=torch.int32, device=device)
    qd = [x.to(device) for x in q]
    outs, keep = [torch.empty_like(x) for x in qd], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            a = nat.PagedAttnArgs(q=qd[i].data_ptr(), q_stride_b=qd[i].stride(0), q_stride_h=qd[i].stride(1), q_stride_s=qd[i].stride(2),
                                  out=outs[i].data_ptr(), o_stride_b=outs[i].stride(0), o_stride_h=outs[i].stride(1),
                                  o_stride_s=outs[i].stride(2), block_table=table.data_ptr(), table_stride=table.stride(0),
                                  seq_lens=lens_dev.data_ptr(), batch=2, num_q_heads=H * rep, q_len=1, causal=1, max_seq_len=2500,
                                  scale=1 / math.sqrt(D))
            ws = torch.empty(int(lib.pace_paged_attn_workspace_for(ctypes.byref(c.pool_desc), ctypes.byref(a))), dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
            keep.append(ws)
            nat.check(lib.pace_paged_attn_decode(ctypes.byref(c.pool_desc), ctypes.byref(a), s.cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        check(outs[i], q[i], k, v, lens, 4, what=f"stream {i}")


def test_the_same_bits_from_call_to_call(device):
    lens, H, rep, D = [3000, 77, 1200], 2, 4, 128
    c, _, _ = filled(device, 4, lens, H, rep, D)
    for S in (1, 9, 100):
        q = rows(5, 3, H * rep, S, D).to(device)
        first = c.attend(q)
        for _ in range(4):
            assert torch.equal(first, c.attend(q))


def test_a_new_window_ends_a_captured_step(device):
    from pace_mi355.llm import KVCacheManager, KVCacheType

    class Cfg:
        num_hidden_layers = 1
        num_attention_heads = 4
        num_key_value_heads = 2

    mgr = KVCacheManager(Cfg(), 64, KVCacheType.PAGED, kv_bits=4)
    x = rows(1, 1, 2, 9, 64).to(device)
    mgr[0].update_cache(x, x, 2)
    k, q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device=device), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=device)
    graph = mgr.capture_decode(lambda: (mgr[0].update_cache(k, k, 2), mgr[0].attend(q))[1], 8)
    graph.replay()
    mgr[0].set_window(4, 1)
    with pytest.raises(RuntimeError, match="spent"):
        graph.replay()
    assert len(mgr) == 10
