"""An attention call that is refused leaves the cache as it was: the step's held-back append and its rotation are still there for the
call that follows."""
import pytest
import torch

from helpers import assert_bits_equal
from test_gpu_walk_shares import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, window, dtype", [(4, None, torch.bfloat16), (16, 20, torch.bfloat16), (16, None, torch.bfloat16), (16, None, torch.float32)])
@pytest.mark.parametrize("rotate", [False, True])
def test_the_next_call_finds_the_step_whole(device, bits, window, dtype, rotate):
    from pace_mi355.llm import PagedKVCache
    from pace_mi355.ops import RotaryEmbedding

    B, H, rep, D, P = 2, 2, 4, 64, 40
    rope = RotaryEmbedding(None, D, 128, 10000.0, dtype=dtype)
    feed = lambda seed, n: [rows(seed + i, B, h, n, D).to(dtype).to(device) for i, h in enumerate((H, H, H * rep))]
    call = lambda at, n: rope(torch.zeros(1, dtype=dtype, device=device), torch.arange(at, at + n, device=device)[None].expand(B, n).contiguous()) if rotate else None
    outs, held = [], []
    for refused in (False, True):
        c = PagedKVCache(64, num_kv_heads=H, n_rep=rep, kv_bits=bits, window=window)
        k, v, q = feed(1, P)
        c.update_cache(k, v, 2, rope=call(0, P))
        c.attend(q)
        k, v, q = feed(11, 1)
        c.update_cache(k, v, 2, rope=call(P, 1))
        if refused:
            with pytest.raises(RuntimeError, match="takes a mask"):
                c.attend(q, torch.zeros(B, 2, 1, P + 1, device=device))
            with pytest.raises(RuntimeError, match="only support the dtypes"):
                c.attend(q, torch.zeros(B, 1, 1, P + 1, dtype=torch.float16, device=device))
            if bits == 4 or window:
                c.partition_tokens = 16
                with pytest.raises(RuntimeError, match="partition_tokens 16"):
                    c.attend(q)
                c.partition_tokens = 0
        outs.append(c.attend(q))
        held.append(c.gather())
    for a, b in zip(held[0], held[1]):
        assert_bits_equal(a, b, "what the cache holds")
    assert_bits_equal(outs[0], outs[1], "the step's output")


@pytest.mark.parametrize("bits, window", [(4, None), (16, 20), (16, None)])
def test_tensors_the_kernels_cannot_read_are_refused(device, bits, window):
    """Tensors of the host, and a kv_start that is not one int32 per sequence."""
    from pace_mi355.llm import PagedKVCache

    B, H, D, P = 2, 2, 64, 40
    c = PagedKVCache(64, num_kv_heads=H, kv_bits=bits, window=window)
    k, q = rows(1, B, H, P, D), rows(2, B, H, 1, D).to(device)
    c.update_cache(k.to(device), k.to(device), 2)
    one = k[:, :, :1].contiguous()
    for a, b in ((one, one.to(device)), (one.to(device), one), (one, one)):
        with pytest.raises(RuntimeError, match="the cache lies on cuda:0"):
            c.update_cache(a, b, 2)
        with pytest.raises(RuntimeError, match="the cache lies on cuda:0"):
            c.append_ragged(a, b, [1, 0])
    with pytest.raises(RuntimeError, match="got a mask on cpu"):
        c.attend(q, torch.zeros(B, 1, 1, P))
    start = torch.tensor([0, 5], dtype=torch.int32)
    wide = torch.zeros(4, dtype=torch.int32, device=device)
    for bad in (start, start.long().to(device), start[:1].to(device), wide[::2]):
        with pytest.raises(RuntimeError, match="kv_start is a contiguous int32 tensor"):
            c.attend(q, kv_start=bad)
    assert c.seq_len == P
    assert torch.equal(c.attend(q, kv_start=start.to(device))[0], c.attend(q)[0])
