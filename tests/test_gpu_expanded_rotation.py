"""Keys and values expanded over heads or sequences by stride 0, with a rotation in a launch of its own: the rotated keys are laid out
anew, and the values are read by their own strides."""
import pytest
import torch

from helpers import assert_bits_equal
from test_gpu_walk_shares import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, window, dtype", [(4, None, torch.bfloat16), (4, 20, torch.bfloat16), (16, 20, torch.bfloat16), (16, None, torch.bfloat16),
                                                 (16, None, torch.float32)])
@pytest.mark.parametrize("over", ["heads", "sequences"])
@pytest.mark.parametrize("T", [1, 40])
def test_expanded_keys_and_values(device, bits, window, dtype, over, T):
    from pace_mi355.llm import PagedKVCache
    from pace_mi355.ops import RotaryEmbedding

    B, D, n_rep = 3, 64, 4
    H = 1 if over == "heads" else 2
    rope = RotaryEmbedding(None, D, 128, 10000.0, dtype=dtype)
    call = rope(torch.zeros(1, dtype=dtype, device=device), torch.arange(T, device=device)[None].expand(B, T).contiguous())
    k, v = (rows(i, B if over == "heads" else 1, H, T, D).to(dtype).to(device) for i in (1, 2))
    q = rows(3, B, H * n_rep, T, D).to(dtype).to(device)
    got = []
    for lay_out in (lambda x: x.contiguous(), lambda x: x):
        c = PagedKVCache(96, num_kv_heads=H, n_rep=n_rep, kv_bits=bits, window=window)
        shape = (B, n_rep, T, D) if over == "heads" else (B, H, T, D)
        c.update_cache(lay_out(k.expand(shape)), lay_out(v.expand(shape)), 2, rope=call)
        got.append((c.attend(q), *c.gather(n_rep=1)))
    for a, b in zip(*got):
        assert_bits_equal(a, b)
