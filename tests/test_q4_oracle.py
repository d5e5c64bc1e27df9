"""The 4-bit row format: properties of the oracle, and refusals that need no GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import q4_ref


def _rows(kind, D=128, n=64):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(n, D, generator=g)
    if kind == "offset":
        x = 100 + 0.01 * x
    elif kind == "tiny":
        x = x * 2.0 ** -20
    elif kind == "wide":
        x = x * torch.exp(4 * torch.randn(D, generator=g))
    elif kind == "equal":
        x = x[:, :1].expand(n, D)
    return x.bfloat16()


@pytest.mark.parametrize("kind", ["plain", "offset", "tiny", "wide", "equal"])
def test_every_value_is_within_half_a_step(kind):
    x = _rows(kind)
    code, s, m = q4_ref.quantise(x)
    assert code.min() >= -8 and code.max() <= 7
    err = (q4_ref.values64(x) - x.double().clamp(-q4_ref.CLAMP, q4_ref.CLAMP)).abs().reshape(-1, 4, 32).numpy()
    # half a step, or where the middle's own rounding (2^-11 of it, 2^-25 below the halves' normal range) moved the codes' span:
    # what then lies outside it is cut by up to that much
    bound = 0.5 * s.astype(np.float64) + np.abs(m.astype(np.float64)) * 2.0 ** -11 + 2.0 ** -25
    assert (err <= bound[..., None]).all()


def test_the_step_is_the_least_that_covers_the_group():
    x = _rows("wide", n=200)
    _, s, _ = q4_ref.quantise(x)
    y = x.double().clamp(-q4_ref.CLAMP, q4_ref.CLAMP).reshape(-1, 4, 32)
    width = (y.amax(-1) - y.amin(-1)).numpy()
    assert (15 * s.astype(np.float64) >= width).all()
    below = np.nextafter(s, np.float16(0)).astype(np.float64)
    assert ((s == 0) | (15 * below < width)).all()


def test_non_finite_values():
    x = torch.randn(2, 64).bfloat16()
    x[0, 3], x[0, 40], x[1, 5] = math.nan, math.inf, -math.inf
    y = x.clone()
    y[0, 3], y[0, 40], y[1, 5] = 0.0, 32768.0, -32768.0
    assert torch.equal(q4_ref.values64(x), q4_ref.values64(y)) and torch.isfinite(q4_ref.values64(x)).all()


def test_a_window_of_the_whole_sequence_is_no_window():
    assert torch.equal(q4_ref.readable(20, 5), q4_ref.readable(20, 5, window=20))
    ok = q4_ref.readable(20, 2, window=3, sinks=2, start=4)
    assert ok[0].nonzero().flatten().tolist() == [4, 5, 16, 17, 18]
    assert ok[1].nonzero().flatten().tolist() == [4, 5, 17, 18, 19]


# ---- refusals (nothing is launched) ----------------------------------------------------------------------------------
def _pool(nat, **kw):
    f = dict(k=1 << 20, v=(1 << 20) + 1280, k_block_stride=20480, k_head_stride=2560, v_block_stride=20480, v_head_stride=2560,
             num_blocks=4, num_kv_heads=8, head_dim=128, block_size=16, elem_bytes=nat.ELEM_Q4)
    f.update(kw)
    return nat.PoolDesc(**f)


def _args(nat, **kw):
    f = dict(q=1 << 20, q_stride_b=4096, q_stride_h=128, q_stride_s=128, out=1 << 20, o_stride_b=4096, o_stride_h=128, o_stride_s=128,
             block_table=16, table_stride=4, seq_lens=16, batch=1, num_q_heads=32, q_len=1, causal=1, max_seq_len=64, scale=0.1)
    f.update(kw)
    return nat.PagedAttnArgs(**f)


@pytest.mark.parametrize("change, text", [
    (dict(head_dim=80), b"head_dim 80 unsupported"),
    (dict(k_head_stride=1264), b"head stride smaller than a slab"),
    (dict(v_head_stride=2568), b"multiples of 16 elements"),
    (dict(k=(1 << 20) + 8), b"16-byte aligned"),
    (dict(block_size=32), b"block_size 32"),
    (dict(elem_bytes=3), b"elem_bytes 3"),
])
def test_pool_refusals(change, text):
    from pace_mi355 import _native as nat

    lib = nat.load()
    pool = _pool(nat, **change)
    assert lib.pace_kv_append(ctypes.byref(pool), 16, 16, 8, 8, 8, 1, 1, 16, None) == -1
    assert text in lib.pace_kv_last_error()
    assert lib.pace_paged_attn_decode(ctypes.byref(pool), ctypes.byref(_args(nat)), None) == -1
    assert text in lib.pace_kv_last_error()


@pytest.mark.parametrize("elem, change, text", [
    (1, dict(window=-1), b"negative window"),
    (1, dict(window=8, sinks=-2), b"negative window"),
    (1, dict(sinks=4), b"come with a window"),
    (2, dict(sinks=4), b"come with a window"),
    (4, dict(window=8), b"a window over an fp32 pool is not supported"),
    (1, dict(q=(1 << 20) + 2), b"q must be 16-byte aligned"),
    (1, dict(scale=0.0), b"softmax scale"),
    (1, dict(partition_tokens=48), b"partition_tokens 48"),
    (2, dict(window=8, partition_tokens=48), b"partition_tokens 48"),
    (1, dict(num_q_heads=31), b"not a multiple of num_kv_heads"),
    (1, dict(max_seq_len=65), b"cannot hold max_seq_len"),
    (1, dict(k_new=1 << 20), b"given together"),
    (1, dict(k_new=1 << 20, v_new=1 << 20, n_new=33), b"1..32 new tokens"),
    (1, dict(workspace=(1 << 20) + 8, workspace_bytes=1 << 20), b"workspace must be 16-byte aligned"),
])
def test_attention_refusals(elem, change, text):
    from pace_mi355 import _native as nat

    lib = nat.load()
    pool = _pool(nat, elem_bytes=elem, v=(1 << 20) + 2560 * 8, k_block_stride=1 << 17, k_head_stride=1 << 13, v_block_stride=1 << 17,
                 v_head_stride=1 << 13)
    assert lib.pace_paged_attn_verify(ctypes.byref(pool), ctypes.byref(_args(nat, **change)), None) == -1
    assert text in lib.pace_kv_last_error()


def test_rope_is_refused_inside_these_launches():
    from pace_mi355 import _native as nat

    lib = nat.load()
    rope = nat.RopeDesc(cos=16, sin=32, table_dtype=1, table_rows=8, rotary_dim=128, interleaved=0)
    for elem, window in ((1, 0), (2, 16)):
        pool = _pool(nat, elem_bytes=elem, k_block_stride=1 << 17, k_head_stride=1 << 13, v_block_stride=1 << 17, v_head_stride=1 << 13)
        args = _args(nat, window=window)
        args.rope = ctypes.pointer(rope)
        assert lib.pace_paged_attn_decode(ctypes.byref(pool), ctypes.byref(args), None) == -1
        assert b"no rotary embedding inside the attention launch" in lib.pace_kv_last_error()
    pool = _pool(nat)
    assert lib.pace_rope_append_paged(ctypes.byref(pool), ctypes.byref(rope), None, None, 0, 0, 0, 0, 16, 16, 8, 8, 8, 1, 1, 16, 1, 16, 0,
                                      None) == -1
    assert b"the pool holds 4-bit rows" in lib.pace_kv_last_error()


def test_copy_between_pools_of_different_kinds_is_refused():
    from pace_mi355 import _native as nat

    lib = nat.load()
    a = _pool(nat)
    b = _pool(nat, elem_bytes=2, k_block_stride=1 << 17, k_head_stride=1 << 13, v_block_stride=1 << 17, v_head_stride=1 << 13)
    assert lib.pace_kv_copy_blocks(ctypes.byref(a), ctypes.byref(b), 16, 1, None) == -1
    assert b"differ in element type" in lib.pace_kv_last_error()


def test_workspace_of_a_call():
    from pace_mi355 import _native as nat

    lib = nat.load()
    pool = _pool(nat)
    need = lambda **kw: int(lib.pace_paged_attn_workspace_for(ctypes.byref(pool), ctypes.byref(_args(nat, **kw))))
    assert need(batch=64, max_seq_len=4096) == 0          # one workgroup per sequence and head fills the GPU
    one = need(batch=1, max_seq_len=4096)
    assert one > 0 and one % (32 * 130 * 4) == 0          # whole partitions of 32 rows of 128 dims, a maximum and a sum
    assert need(batch=1, max_seq_len=1 << 20, window=256, sinks=4) < one  # as much as the window takes, whatever the length
    assert need(batch=0) == 0 and need(num_q_heads=31) == 0


def test_cache_options():
    from pace_mi355.llm import KVCacheManager, KVCacheType, PagedKVCache

    with pytest.raises(ValueError, match="kv_bits must be 4 or 16"):
        PagedKVCache(64, kv_bits=8)
    for bad in (dict(window=-1), dict(sinks=3), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            PagedKVCache(64, **bad)

    class Cfg:
        num_hidden_layers = 2
        num_attention_heads = 8
        num_key_value_heads = 2

    mgr = KVCacheManager(Cfg(), 64, KVCacheType.PAGED, kv_bits=4, window=16, sinks=2)
    assert [(c.kv_bits, c.window, c.sinks) for c in (mgr[0], mgr[1])] == [(4, 16, 2)] * 2
    mgr[1].set_window(None)
    assert (mgr[1].window, mgr[1].sinks) == (0, 0) and mgr[0].window == 16
