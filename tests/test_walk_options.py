"""Options of the 4-bit cache and of the window, and sizes a launch is asked about, that need no GPU."""
import ctypes
import os
import subprocess
import sys

import pytest

from test_q4_oracle import _args, _pool


def need(elem_bytes=1, **kw):
    """The scratch the library asks for."""
    from pace_mi355 import _native as nat

    pool = _pool(nat) if elem_bytes == 1 else _pool(nat, elem_bytes=elem_bytes, k_block_stride=1 << 17, k_head_stride=1 << 13,
                                                    v_block_stride=1 << 17, v_head_stride=1 << 13)
    return int(nat.load().pace_paged_attn_workspace_for(ctypes.byref(pool), ctypes.byref(_args(nat, **kw))))


def test_a_cut_that_is_no_multiple_of_32_needs_nothing():
    """(In a process of its own, which a division by zero would end.)"""
    code = ("from test_walk_options import need\n"
            "for elem, window in ((1, 0), (2, 64)):\n"
            "  for tokens in (1, 16, 31, 33, 48, -1, -32):\n"
            "    for batch, q_len in ((1, 1), (8, 1), (1, 9), (3, 100)):\n"
            "      got = need(elem, batch=batch, q_len=q_len, max_seq_len=4096, partition_tokens=tokens, window=window)\n"
            "      assert got == 0, (elem, tokens, batch, q_len, got)\n"
            "print('done')")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=env, cwd=os.path.dirname(os.path.abspath(__file__)))
    assert r.returncode == 0 and r.stdout.split() == ["done"], f"exit status {r.returncode}: {r.stderr[-500:]}"


def test_a_cut_is_the_longest_run_of_a_workgroup():
    """Nothing is cut that fits, however many sequences there are, and no workgroup takes the sequences of others besides."""
    piece = 8 * 2 * 4 * 130 * 4  # two partial results of 4 query rows for each of 8 KV heads: 128 dims, a maximum and a sum
    for batch in (1, 2, 64):
        for longest in (1, 100, 4096):
            assert need(batch=batch, max_seq_len=longest, partition_tokens=4096) == 0, (batch, longest)
        assert need(batch=batch, max_seq_len=8192, partition_tokens=4096) == 2 * batch * piece
        assert need(batch=batch, max_seq_len=8192, partition_tokens=1 << 20) == 0
        assert need(2, batch=batch, max_seq_len=1 << 17, partition_tokens=4096, window=2048, sinks=4) == 0  # the window fits


class _Cfg:
    num_hidden_layers = 2
    num_attention_heads = 8
    num_key_value_heads = 2


@pytest.mark.parametrize("cache_type", ["dynamic", "bmc"])
@pytest.mark.parametrize("option", [dict(kv_bits=4), dict(window=16), dict(window=16, sinks=2)])
def test_caches_that_store_no_blocks_refuse_these_options(cache_type, option):
    """They keep the model's dtype and their attention reads everything: taken silently, the options would change nothing."""
    from pace_mi355.llm import KVCacheManager

    with pytest.raises(ValueError, match="paged cache"):
        KVCacheManager(_Cfg(), 64, cache_type, **option)
    assert len(KVCacheManager(_Cfg(), 64, cache_type, kv_bits=16, window=None, sinks=0, num_blocks=8).cache_objects) == 2


@pytest.mark.parametrize("huge", [1 << 31, (1 << 32) + 5, 1 << 40])
def test_a_window_wider_than_any_sequence_stays_one(huge):
    """Positions are 32-bit numbers; a window or a count of sinks past them must not wrap around to a small one."""
    from pace_mi355 import _native as nat
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(64, window=huge, sinks=huge)
    a = nat.PagedAttnArgs(window=c.window, sinks=c.sinks)
    assert a.window == a.sinks == (1 << 31) - 1
