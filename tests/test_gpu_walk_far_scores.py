"""Masks filled with large finite numbers, and scores far from 0: the softmax of the kernels behind a 4-bit cache and behind a window
stays one (its weights sum to 1) wherever the scores lie."""
import pytest
import torch

from oracle import q4_ref
from test_gpu_walk_shares import filled, rows

pytestmark = pytest.mark.gpu

FILLS = [-1e4, -65504.0, -1e6, -1e7, -1e8, -1e9, -1e10, -1e12, -1e20, -1e29]


def cache_of(device, bits, H, rep, D, L, B, v_rows):
    from pace_mi355.llm import PagedKVCache

    c = PagedKVCache(L + 16, num_kv_heads=H, n_rep=rep, kv_bits=bits, window=None if bits == 4 else L)
    k = rows(1, B, H, L, D)
    c.append_ragged(k.to(device), v_rows.to(device), [L] * B)
    return c, k


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("S, D", [(1, 128), (9, 64), (70, 128), (33, 256)])
@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_masks_of_any_fill(device, bits, S, D, fill, dtype):
    """Left padding: whole units at the fill value come first, and the rows of the padding itself have nothing else."""
    B, H, rep, L, pads = 3, 2, 2, 200, (0, 70, 199)
    v = rows(2, B, H, L, D)
    c, k = cache_of(device, bits, H, rep, D, L, B, v)
    q = rows(3, B, H * rep, S, D)
    t, pos = torch.arange(L)[None], (L - S + torch.arange(S))[:, None]
    mask = torch.stack([torch.where((t <= pos) & (t >= p), 0.0, fill) for p in pads])[:, None].to(dtype)
    out = c.attend(q.to(device), mask.to(device)).double().cpu()
    assert torch.isfinite(out).all()
    held = q4_ref.values64 if bits == 4 else (lambda x: x.double())
    for b in range(B):
        real = (mask[b, 0] == 0).any(-1)  # rows with an unmasked column: there a weight of exp(fill) is 0 in any precision
        ok = q4_ref.readable(L, S, 0 if bits == 4 else L, 0, causal=False)
        ref, parts = q4_ref.attention64(q[b], held(k[b]), held(v[b]), ok, mask[b, 0].float())
        near = (out[b] - ref).abs() <= q4_ref.error_bound(ref, parts, bits)
        assert bool(near[:, real].all()), f"sequence {b}"


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("S, D", [(1, 128), (9, 64), (70, 128), (33, 256), (70, 96)])
@pytest.mark.parametrize("fill", [None] + FILLS)
@pytest.mark.parametrize("split", [0, 64])
def test_the_weights_sum_to_one(device, bits, S, D, fill, split):
    """All values alike: any weights that sum to 1 give them back.  Rows that are masked throughout, at any fill value, and
    (without a mask) scores of 1 to 10^9."""
    B, H, rep, L = 2, 2, 2, 300
    each = (1.0 + torch.arange(D) // 32).bfloat16()  # alike within a group of 32 dims too: exact in the 4-bit form
    c, _ = cache_of(device, bits, H, rep, D, L, B, each.expand(B, H, L, D).contiguous())
    c.partition_tokens = split
    want = each.double()
    if fill is not None:
        q = rows(3, B, H * rep, S, D)
        for m in (torch.full((B, 1, S, L), fill), torch.full((1, 1, 1, L), fill).bfloat16()):
            out = c.attend(q.to(device), m.to(device)).double().cpu()
            # as many equal or smaller weights above as below the fraction: sums of 300 terms, and the output's rounding to bf16
            assert bool(((out - want).abs() <= (2.0 ** -8 + 300 * 2.0 ** -24) * want).all()), f"{out[0, 0, 0, :3]} at {fill}"
        return
    for scale in (1.0, 1e3, 1e5, 1e6, 1e7, 1e8, 1e9):
        q = (rows(3, B, H * rep, S, D) * scale).bfloat16()
        out = c.attend(q.to(device)).double().cpu()
        assert bool(((out - want).abs() <= (2.0 ** -8 + 300 * 2.0 ** -24) * want).all()), f"{out[0, 0, 0, :3]} at {scale}"


@pytest.mark.parametrize("bits", [4, 16])
def test_one_far_score_takes_it_all(device, bits):
    """One key points the query's way, the others away from it, at growing lengths: the row becomes its value."""
    B, H, D, L = 1, 1, 64, 200
    c, k, v = filled(device, bits, [L], H, 1, D, None if bits == 4 else L)
    c.truncate([L])
    k = torch.full((B, H, L, D), -1.0).bfloat16()
    k[0, 0, 77] = 1.0
    c.append_ragged(k.to(device), v.to(device), [L])
    held = q4_ref.values64 if bits == 4 else (lambda x: x.double())
    for scale in (1e2, 1e4, 1e6, 1e8, 1e12):
        out = c.attend(torch.full((B, H, 1, D), scale).bfloat16().to(device)).double().cpu()
        want = held(v)[0, 0, 77]
        # the value to a half (4-bit pools), the output to bf16
        assert bool(((out[0, 0, 0] - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * want.abs() + 2.0 ** -24).all()), scale
