"""A frozen step (``FixedStep``) over a 4-bit cache and through a window: the cache's own options reach the launch."""

import pytest
import torch

from test_gpu_walk_shares import check, filled, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, window, sinks", [(4, None, 0), (4, 50, 3), (16, 50, 3)])
@pytest.mark.parametrize("S", [1, 6])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("partition", [0, 64])
def test_a_frozen_step_is_the_caches_own(device, bits, window, sinks, S, fused, partition):
    from pace_mi355.utils.fixed_step import FixedStep

    lens, H, rep, D = [700, 33, 190], 2, 4, 64
    c, k, v = filled(device, bits, lens, H, rep, D, window, sinks)
    kn, vn, q = rows(7, 3, H, S, D), rows(8, 3, H, S, D), rows(9, 3, H * rep, S, D)
    step = FixedStep(torch, c, q.to(device), kn.to(device), vn.to(device), partition=partition, fused=fused)
    assert "walk_" in step.kernel
    after = [n + S for n in lens]
    kk, vv = (torch.zeros(3, H, max(after), D, dtype=torch.bfloat16) for _ in range(2))
    for b, n in enumerate(lens):
        for x, old, new in ((kk, k, kn), (vv, v, vn)):
            x[b, :, :n], x[b, :, n:n + S] = old[b, :, :n], new[b]
    for _ in range(2):  # the same positions every step
        step()
        check(step.out, q, kk, vv, after, bits, window or 0, sinks, what=f"{bits} S={S} fused {fused}")


def test_a_mask_tensor_and_a_window(device):
    from pace_mi355.utils.fixed_step import FixedStep

    lens, H, rep, D, S = [120, 120], 2, 2, 64, 5
    c, k, v = filled(device, 16, lens, H, rep, D, 30, 2)
    kn, vn, q = rows(7, 2, H, S, D), rows(8, 2, H, S, D), rows(9, 2, H * rep, S, D)
    t, pos = torch.arange(125)[None], (120 + torch.arange(S))[:, None]
    mask = torch.stack([torch.where((t <= pos) & (t >= p), 0.0, torch.finfo(torch.bfloat16).min) for p in (0, 100)])[:, None].bfloat16()
    step = FixedStep(torch, c, q.to(device), kn.to(device), vn.to(device), mask=mask.to(device))
    step()
    kk, vv = torch.cat([k, kn], 2), torch.cat([v, vn], 2)
    check(step.out, q, kk, vv, [125, 125], 16, 30, 2, mask=mask, what="mask")


def test_a_rotation_that_no_launch_takes_is_refused(device):
    """Over these caches no launch rotates: neither the attention nor the append of a 4-bit pool."""
    from pace_mi355.ops import RotaryEmbedding
    from pace_mi355.utils.fixed_step import FixedStep

    kn, q = rows(7, 1, 2, 1, 64).to(device), rows(9, 1, 8, 1, 64).to(device)
    rope = RotaryEmbedding(None, 64, 256, 10000.0)(q, torch.zeros(1, 1, dtype=torch.int64, device=device))
    for bits, window in ((4, None), (16, 20)):
        c, _, _ = filled(device, bits, [40], 2, 4, 64, window)
        with pytest.raises(RuntimeError, match="no rotary embedding inside the attention launch"):
            FixedStep(torch, c, q, kn, kn, rope=rope.desc())()
