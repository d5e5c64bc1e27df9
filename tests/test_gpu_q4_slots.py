"""Append by slot into a 4-bit pool through the C ABI: slots in any order and from several sequences, missing and foreign ones,
tokens that share a dword of V with tokens of other workgroups and of earlier calls."""
import ctypes

import pytest
import torch

from helpers import assert_bits_equal
from oracle import q4_ref

pytestmark = pytest.mark.gpu


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def order_of(kind, total, count, g):
    """`count` different slots of `total`."""
    if kind == "shuffled":
        return torch.randperm(total, generator=g)[:count]
    if kind == "backwards":
        return torch.arange(count).flip(0) + 3
    if kind == "shifted":
        return torch.arange(count) + 5
    return torch.arange(count) * (total // count)  # strided


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("kind", ["shuffled", "backwards", "shifted", "strided"])
@pytest.mark.parametrize("B, T", [(1, 1), (3, 7), (2, 50)])
def test_slots_in_any_order(device, D, kind, B, T):
    from pace_mi355 import _native as nat

    lib, H, nb = nat.load(), 2, 13
    total = nb * 16
    pool = torch.zeros(nb, H, 2, 10 * D, dtype=torch.uint8, device=device)
    desc = nat.PoolDesc(k=pool.data_ptr(), v=pool.data_ptr() + 10 * D, k_block_stride=pool.stride(0), k_head_stride=pool.stride(1),
                        v_block_stride=pool.stride(0), v_head_stride=pool.stride(1), num_blocks=nb, num_kv_heads=H, head_dim=D, block_size=16,
                        elem_bytes=nat.ELEM_Q4)
    held = torch.zeros(2, H, total, D, dtype=torch.bfloat16)  # what the slots stand for
    g = torch.Generator().manual_seed(B * T + D)
    for call, missing in enumerate((False, True, True)):
        k, v = rows(10 + call, B, H, T, D), rows(20 + call, B, H, T, D)
        slots = order_of(kind, total, B * T, g).reshape(B, T)
        if missing:  # none, and slots that lie outside the pool
            away = torch.rand(B, T, generator=g) < 0.4
            slots = torch.where(away, torch.where(torch.rand(B, T, generator=g) < 0.5, -1, total + slots), slots)
        kd, vd, sd = k.to(device), v.to(device), slots.contiguous().to(device)
        nat.check(lib.pace_kv_append(ctypes.byref(desc), kd.data_ptr(), vd.data_ptr(), kd.stride(0), kd.stride(1), kd.stride(2), B, T, sd.data_ptr(),
                                     nat.current_stream_ptr()))
        for b in range(B):
            for t in range(T):
                if 0 <= slots[b, t] < total:
                    held[0, :, slots[b, t]], held[1, :, slots[b, t]] = q4_ref.values_bf16(k[b, :, t]), q4_ref.values_bf16(v[b, :, t])
        out = torch.empty(2, 1, H, total, D, dtype=torch.bfloat16, device=device)
        table, lens = torch.arange(nb, dtype=torch.int32, device=device), torch.tensor([total], dtype=torch.int32, device=device)
        nat.check(lib.pace_kv_gather(ctypes.byref(desc), table.data_ptr(), nb, lens.data_ptr(), 0, 1, 1, out[0].data_ptr(), out[1].data_ptr(),
                                     out.stride(1), out.stride(2), total, 0, nat.current_stream_ptr()))
        assert_bits_equal(out[0, 0].cpu(), held[0], f"K {kind} call {call}")
        assert_bits_equal(out[1, 0].cpu(), held[1], f"V {kind} call {call}")
