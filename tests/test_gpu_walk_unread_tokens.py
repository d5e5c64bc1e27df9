"""Attention through a window over a 16-bit pool in several row groups per sequence: what only later groups read may hold
anything without touching the rows of earlier ones."""
import math

import pytest
import torch

from oracle import q4_ref
from test_gpu_walk_groups import WHOLE, name_of
from test_gpu_walk_shares import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S, rep, D, split", [(8, 4, 128, 0), (5, 8, 64, 0), (12, 2, 96, 0), (10, 4, 256, 0), (150, 2, 64, 0), (90, 4, 128, 0),
                                               (50, 4, 256, 0), (150, 2, 64, WHOLE), (90, 4, 128, WHOLE), (80, 2, 96, WHOLE), (50, 4, 256, WHOLE)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_tokens_that_only_later_groups_read(device, S, rep, D, split, bad):
    from pace_mi355.llm import PagedKVCache

    H, L, window, sinks = 2, S + 37, 24, 3
    c = PagedKVCache(L + 16, num_kv_heads=H, n_rep=rep, window=window, sinks=sinks)
    c.partition_tokens = split
    k, v, q = rows(1, 1, H, L, D), rows(2, 1, H, L, D), rows(3, 1, H * rep, S, D)
    name = name_of_first_call(c, k, v, q, device, rep)
    group = 16 if "walk_attn" in name else (64 if f"<16, {D}, 1," in name else 128)
    assert S * rep > group, f"{name}: one group only"
    whole = group // rep  # query tokens that lie in the first group with all their heads
    last = (group - 1) // rep  # the last query token that has a row in it
    late = L - S + last + 1  # tokens from here on are read by later groups only
    k[:, :, late:], v[:, :, late:] = bad, bad
    c.append_ragged(k.to(device), v.to(device), [L])
    out = c.attend(q.to(device)).double().cpu()[0, :, :whole]
    # (oracle: the same rows of a sequence that ends before the bad tokens)
    ok = q4_ref.readable(L, S, window, sinks)[:whole, :late]
    ref, parts = q4_ref.attention64(q[0, :, :whole], k[0, :, :late].double(), v[0, :, :late].double(), ok)
    assert torch.isfinite(out).all(), f"{name}: a later token reached rows that do not read it"
    assert bool(((out - ref).abs() <= q4_ref.error_bound(ref, parts, 16)).all()), name


def name_of_first_call(c, k, v, q, device, rep):
    """The kernel that serves a sequence of this length; the cache is empty again afterwards."""
    L = k.shape[2]
    c.append_ragged(torch.zeros_like(k).to(device), torch.zeros_like(v).to(device), [L])
    if c.partition_tokens:
        c.attend(q.to(device))  # (the library is asked with partition_tokens 0 below: named by the rows alone here)
        rows_, D = q.shape[2] * rep, k.shape[3]
        name = "walk_attn" if rows_ <= 16 else (f"<16, {D}, 1," if rows_ <= 64 or D == 256 else f"<16, {D}, 2,")
    else:
        name = name_of(c, [L], q.shape[1], q.shape[2])
    c.truncate([L])
    return name
