"""Decode steps captured with a rotary embedding where the rotation runs in launches of its own: over a 4-bit cache, through a
window, over an fp32 pool."""
import pytest
import torch

from oracle import q4_ref

pytestmark = pytest.mark.gpu


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def bound_of(ref, parts, bits):
    if bits != 32:
        return q4_ref.error_bound(ref, parts, bits)
    spread, amp, _ = parts  # nothing is rounded below single precision: the last term of error_bound, and the output's rounding
    return 2.0 ** -23 * ref.abs() + spread * 2.0 ** -14 * (1 + amp) + 1e-30


@pytest.mark.parametrize("bits, window, sinks", [(4, None, 0), (4, 12, 2), (16, 12, 2), (32, None, 0)])
@pytest.mark.parametrize("T", [1, 9])
def test_a_captured_step_rotates_its_queries(device, bits, window, sinks, T):
    from pace_mi355.llm import KVCacheManager, KVCacheType
    from pace_mi355.ops import RotaryEmbedding

    class Cfg:
        num_hidden_layers = 2
        num_attention_heads = 8
        num_key_value_heads = 2

    B, H, rep, D, P, steps = 2, 2, 4, 64, 21, 4
    dtype = torch.float32 if bits == 32 else torch.bfloat16
    mgr = KVCacheManager(Cfg(), 96, KVCacheType.PAGED, kv_bits=4 if bits == 4 else 16, window=window, sinks=sinks)
    rope = RotaryEmbedding(None, D, 256, 10000.0, dtype=dtype)
    held = [([], []) for _ in range(2)]  # per layer: the rotated keys, the values

    def feed(layer, seed, n, at):
        """New rows of a layer; remembers what the cache should then hold.  Returns k, v, q and the rotated q."""
        k, v, q = (rows(seed + i, B, h, n, D).to(dtype) for i, h in enumerate((H, H, H * rep)))
        call = rope(q.to(device), torch.arange(at, at + n, device=device)[None].expand(B, n).contiguous())
        qr, kr = call(q.to(device), k.to(device))
        held[layer][0].append(kr.cpu())
        held[layer][1].append(v)
        return k, v, q, qr.cpu(), call

    def verify(layer, qr, out, what):
        k, v = (torch.cat(x, 2) for x in held[layer])
        out = out.double().cpu()
        value = q4_ref.values64 if bits == 4 else (lambda x: x.double())
        ok = q4_ref.readable(k.shape[2], qr.shape[2], window or 0, sinks)
        for b in range(B):
            ref, parts = q4_ref.attention64(qr[b], value(k[b]), value(v[b]), ok)
            worst = float(((out[b] - ref).abs() / bound_of(ref, parts, bits)).max())
            assert worst <= 1.0, f"{what}, layer {layer}, sequence {b}: {worst:.2f} of the bound"

    for layer in range(2):
        k, v, q, qr, call = feed(layer, 100 * layer, P, 0)
        mgr[layer].update_cache(k.to(device), v.to(device), 2, rope=call)
        verify(layer, qr, mgr[layer].attend(q.to(device)), "prompt")
    static = [[torch.zeros(B, h, T, D, dtype=dtype, device=device) for h in (H, H, H * rep)] for _ in range(2)]
    step_call = rope(static[0][2], torch.arange(P, P + T, device=device)[None].expand(B, T).contiguous())

    def step():
        out = []
        for layer in range(2):
            k, v, q = static[layer]
            mgr[layer].update_cache(k, v, 2, rope=step_call)
            out.append(mgr[layer].attend(q))
        return out

    graph = mgr.capture_decode(step, steps)
    for i in range(steps):
        at, rotated = P + i * T, []
        for layer in range(2):
            k, v, q, qr, call = feed(layer, 1000 + 100 * i + 10 * layer, T, at)
            for to, x in zip(static[layer], (k, v, q)):
                to.copy_(x)
            rotated.append(qr)
        step_call.rows.copy_(call.rows)
        got = graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            verify(layer, rotated[layer], got[layer], f"replay {i}")
    graph.close()
    # and step by step from there
    at = P + steps * T
    for layer in range(2):
        k, v, q, qr, call = feed(layer, 9000 + 10 * layer, 1, at)
        mgr[layer].update_cache(k.to(device), v.to(device), 2, rope=call)
        verify(layer, qr, mgr[layer].attend(q.to(device)), "a step after the graph")
