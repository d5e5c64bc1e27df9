"""Masks filled with large finite numbers over the bf16 and fp32 pools and in the dense operator: what a padded prompt's rows read
comes out the same at any fill value."""
import pytest
import torch

from oracle import q4_ref
from test_gpu_captured_rope import bound_of
from test_gpu_walk_far_scores import FILLS

pytestmark = pytest.mark.gpu


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("S, D", [(1, 128), (9, 64), (70, 128), (300, 128), (33, 256), (200, 96)])
@pytest.mark.parametrize("fill", FILLS + [-1e30])
@pytest.mark.parametrize("where", ["paged", "dense"])
def test_padding_masks_of_any_fill(device, bits, S, D, fill, where):
    """Whole units at the fill value come first, and the rows of the padding itself have nothing else."""
    from pace_mi355.llm import PagedKVCache
    import pace_mi355.ops  # noqa: F401  (registers torch.ops.pace)

    B, H, rep, L, pads = 3, 2, 2, 400, (0, 131, 399)
    dtype = torch.float32 if bits == 32 else torch.bfloat16
    k, v, q = (rows(1 + i, B, h, n, D).to(dtype) for i, (h, n) in enumerate(((H, L), (H, L), (H * rep, S))))
    t, pos = torch.arange(L)[None], (L - S + torch.arange(S))[:, None]
    mask = torch.stack([torch.where((t <= pos) & (t >= p), 0.0, fill) for p in pads])[:, None].to(dtype)
    if where == "paged":
        c = PagedKVCache(L + 16, num_kv_heads=H, n_rep=rep)
        c.append_ragged(k.to(device), v.to(device), [L] * B)
        out = c.attend(q.to(device), mask.to(device))
    else:
        ke, ve = (x.repeat_interleave(rep, 1).contiguous().to(device) for x in (k, v))
        out = torch.ops.pace.attention(q.to(device), ke, ve, mask.to(device), False)
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    for b in range(B):
        real = (mask[b, 0] == 0).any(-1)  # rows with an unmasked column: there a weight of exp(fill) is 0 in any precision
        ref, parts = q4_ref.attention64(q[b], k[b].double(), v[b].double(), q4_ref.readable(L, S, causal=False), mask[b, 0].float())
        assert bool(((out[b] - ref).abs() <= bound_of(ref, parts, bits))[:, real].all()), f"sequence {b}"
        each = out[b][:, ~real]  # the others: an average of values, with whatever weights
        lo, hi = (x.repeat_interleave(rep, 0)[:, None] for x in (v[b].double().amin(1), v[b].double().amax(1)))
        slack = 2.0 ** -7 * torch.maximum(lo.abs(), hi.abs())  # weights and output to bf16: 2^-8 each
        assert bool(((each >= lo - slack) & (each <= hi + slack)).all())
