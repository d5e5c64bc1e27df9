"""Steps run one by one while a captured decode step lives: they end it, and are right."""
import pytest
import torch

from oracle import q4_ref
from test_gpu_captured_rope import bound_of, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, window", [(4, None), (4, 10), (16, 10), (16, None), (32, None)])
@pytest.mark.parametrize("replays", [0, 2])
def test_steps_after_a_capture(device, bits, window, replays):
    from pace_mi355.llm import KVCacheManager, KVCacheType

    class Cfg:
        num_hidden_layers = 2
        num_attention_heads = 8
        num_key_value_heads = 2

    B, H, rep, D, P = 2, 2, 4, 64, 30
    dtype = torch.float32 if bits == 32 else torch.bfloat16
    mgr = KVCacheManager(Cfg(), 96, KVCacheType.PAGED, kv_bits=4 if bits == 4 else 16, window=window)
    held = [([], []) for _ in range(2)]
    static = [[torch.zeros(B, h, 1, D, dtype=dtype, device=device) for h in (H, H, H * rep)] for _ in range(2)]

    def feed(layer, seed, n):
        k, v, q = (rows(seed + i, B, h, n, D).to(dtype) for i, h in enumerate((H, H, H * rep)))
        held[layer][0].append(k)
        held[layer][1].append(v)
        return k, v, q

    def verify(layer, q, out, what):
        k, v = (torch.cat(x, 2) for x in held[layer])
        value = q4_ref.values64 if bits == 4 else (lambda x: x.double())
        ok = q4_ref.readable(k.shape[2], q.shape[2], window or 0)
        for b in range(B):
            ref, parts = q4_ref.attention64(q[b], value(k[b]), value(v[b]), ok)
            worst = float(((out[b].double().cpu() - ref).abs() / bound_of(ref, parts, bits)).max())
            assert worst <= 1.0, f"{what}, layer {layer}, sequence {b}: {worst:.2f} of the bound"

    def step():
        out = []
        for layer in range(2):
            k, v, q = static[layer]
            mgr[layer].update_cache(k, v, 2)
            out.append(mgr[layer].attend(q))
        return out

    for layer in range(2):
        k, v, q = feed(layer, 100 * layer, P)
        mgr[layer].update_cache(k.to(device), v.to(device), 2)
        mgr[layer].attend(q.to(device))
    graph = mgr.capture_decode(step, 8)
    for i in range(replays + 3):
        fresh = [feed(layer, 1000 + 100 * i + 10 * layer, 1) for layer in range(2)]
        for layer in range(2):
            for to, x in zip(static[layer], fresh[layer]):
                to.copy_(x)
        out = graph.replay() if i < replays else step()
        torch.cuda.synchronize()
        for layer in range(2):
            verify(layer, fresh[layer][2], out[layer], f"{'replay' if i < replays else 'step'} {i}")
    with pytest.raises(RuntimeError, match="spent"):
        graph.replay()
    assert len(mgr) == P + replays + 3
