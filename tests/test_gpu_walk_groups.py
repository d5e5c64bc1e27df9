"""Attention over the 4-bit cache and through a window, by the size of the row groups: 16, 64 and 128 rows, each with several
groups per sequence, with and without a mask, windows that begin inside a group, and the sizes at which the library picks each."""
import pytest
import torch

from test_gpu_walk_shares import check, filled, rows

pytestmark = pytest.mark.gpu

WHOLE = 1 << 20  # partition_tokens: the largest groups for the rows, each walked whole


def name_of(cache, lens, hq, S):
    from pace_mi355 import _native as nat

    a = nat.PagedAttnArgs(batch=len(lens), num_q_heads=hq, q_len=S, causal=1, max_seq_len=max(lens), scale=1.0, window=cache.window, sinks=cache.sinks)
    q = torch.zeros(len(lens), hq, S, cache.head_dim, dtype=torch.bfloat16, device="cuda")
    table, lens_dev = cache.state.device_table(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    for x in ("q", "o"):
        for s, n in zip("bhs", q.stride()):
            setattr(a, f"{x}_stride_{s}", n)
    a.q = a.out = q.data_ptr()
    a.block_table, a.table_stride, a.seq_lens = table.data_ptr(), table.stride(0), lens_dev.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    return nat.kernel_name(cache.pool_desc, a)


@pytest.mark.parametrize("bits, window, sinks", [(4, None, 0), (4, 40, 3), (16, 100, 5), (16, 1, 0)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("S", [5, 17, 90, 200])
@pytest.mark.parametrize("split", [0, WHOLE])
def test_groups_of_every_size(device, bits, window, sinks, D, S, split):
    lens = [S, 333 + S, 0, 31, 500]
    c, k, v = filled(device, bits, lens, 2, 3, D, window, sinks)
    c.partition_tokens = split
    q = rows(9, 5, 6, S, D)
    check(c.attend(q.to(device)), q, k, v, lens, bits, window or 0, sinks, what=f"{bits} D={D} S={S} window {window}")


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("S, D", [(6, 128), (30, 64), (100, 96), (150, 128), (40, 256)])
@pytest.mark.parametrize("split", [0, WHOLE])
def test_masks_by_group(device, bits, S, D, split):
    """Left padding, as models hand it on, over several groups of rows."""
    L, pads = 400, (0, 77, 399)
    c, k, v = filled(device, bits, [L] * 3, 2, 2, D, None if bits == 4 else L)
    c.partition_tokens = split
    t, pos = torch.arange(L)[None], (L - S + torch.arange(S))[:, None]
    mask = torch.stack([torch.where((t <= pos) & (t >= p), 0.0, torch.finfo(torch.bfloat16).min) for p in pads])[:, None]
    q = rows(9, 3, 4, S, D)
    for m in (mask, mask.bfloat16()):
        check(c.attend(q.to(device), m.to(device)), q, k, v, [L] * 3, bits, 0 if bits == 4 else L, mask=m, what=f"{bits} S={S} {m.dtype}")


@pytest.mark.parametrize("batch, S, name", [(1, 200, "walk_attn_kernel<4, 64,"), (1, 512, "walk_rows_kernel<4, 64, 1,"), (2, 512, "walk_rows_kernel<4, 64, 2,")])
def test_prompts_by_the_rule(device, batch, S, name):
    lens = [S] * batch
    c, k, v = filled(device, 4, lens, 8, 4, 64)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert name in name_of(c, lens, 32, S)
    q = rows(9, batch, 32, S, 64)
    check(c.attend(q.to(device)), q, k, v, lens, 4, what=name)
