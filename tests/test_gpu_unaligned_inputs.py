"""Key/value states and queries that begin at any element: rows of a larger tensor, handed on as views."""
import pytest
import torch

from helpers import assert_bits_equal
from test_gpu_walk_shares import rows

pytestmark = pytest.mark.gpu


def shifted(x, device, by=1):
    """The same tensor, contiguous, `by` elements behind a 16-byte border."""
    room = torch.empty(x.numel() + 16, dtype=x.dtype, device=device)
    out = room[by:by + x.numel()].view(x.shape)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out.copy_(x)


@pytest.mark.parametrize("bits, window, dtype", [(4, None, torch.bfloat16), (16, 20, torch.bfloat16), (16, None, torch.bfloat16), (16, None, torch.float32)])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("T", [1, 40])
def test_the_same_bits_from_any_address(device, bits, window, dtype, rotate, T):
    from pace_mi355.llm import PagedKVCache
    from pace_mi355.ops import RotaryEmbedding

    B, H, rep, D, P = 2, 2, 4, 64, 21
    rope = RotaryEmbedding(None, D, 128, 10000.0, dtype=dtype)
    call = lambda at, n: rope(torch.zeros(1, dtype=dtype, device=device), torch.arange(at, at + n, device=device)[None].expand(B, n).contiguous()) if rotate else None
    got = []
    for place in (lambda x: x.to(device), lambda x: shifted(x, device)):
        c = PagedKVCache(96, num_kv_heads=H, n_rep=rep, kv_bits=bits, window=window)
        for seed, at, n in ((1, 0, P), (11, P, T)):
            k, v, q = (place(rows(seed + i, B, h, n, D).to(dtype)) for i, h in enumerate((H, H, H * rep)))
            c.update_cache(k, v, 2, rope=call(at, n))
            out = c.attend(q)
        k, v = (place(rows(31 + i, B, H, 3, D).to(dtype)) for i in range(2))
        c.append_ragged(k, v, [3, 1])
        got.append((out, *c.gather()))
    for a, b in zip(*got):
        assert_bits_equal(a, b)
