"""Masks of fewer columns than a sequence has tokens, over a 4-bit pool and through a window: a token without a column is read by no
row, also by one that its columns leave nothing but their lowest values, and may hold anything."""
import math

import pytest
import torch

from oracle import q4_ref
from test_gpu_walk_groups import WHOLE
from test_gpu_walk_shares import filled, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, window, sinks", [(4, None, 0), (4, 9, 2), (16, 9, 2), (16, 500, 0)])
@pytest.mark.parametrize("S, D", [(1, 128), (6, 64), (40, 96), (150, 128), (50, 256)])
@pytest.mark.parametrize("missing", [3, 40, 150])
@pytest.mark.parametrize("split", [0, 64, WHOLE])
def test_tokens_without_a_column_are_not_read(device, bits, window, sinks, S, D, missing, split):
    B, H, rep, L = 2, 2, 2, 170
    lens, columns = [L, L - 5], L - missing
    c, k, v = filled(device, bits, lens, H, rep, D, window, sinks)
    if bits == 16:  # (a 4-bit pool holds finite values only)
        k[:, :, columns:], v[:, :, columns:] = math.nan, math.inf
        c.truncate(lens)
        c.append_ragged(k.to(device), v.to(device), lens)
    c.partition_tokens = split
    q = rows(9, B, H * rep, S, D)
    low = torch.finfo(torch.bfloat16).min
    mask = 0.1 * torch.randn(B, 1, S, columns, generator=torch.Generator().manual_seed(4))
    mask[0, 0, : (S + 1) // 2] = low  # nothing but the lowest value: these rows are averages
    mask[1, 0, :, : columns // 2] = -math.inf
    for m in (mask, mask.bfloat16()):
        out = c.attend(q.to(device), m.to(device)).double().cpu()
        assert torch.isfinite(out).all()
        held = q4_ref.values64 if bits == 4 else (lambda x: x.double())
        for b, n in enumerate(lens):
            seen = min(n, columns)
            ok = q4_ref.readable(n, S, window or 0, sinks, causal=False)[:, :seen]
            ref, parts = q4_ref.attention64(q[b], held(k[b, :, :seen]), held(v[b, :, :seen]), ok, m[b, 0, :, :seen].float())
            worst = float(((out[b] - ref).abs() / q4_ref.error_bound(ref, parts, bits)).max())
            assert worst <= 1.0, f"sequence {b}: {worst:.2f} of the bound"
