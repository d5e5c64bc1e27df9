"""Oracle of the 4-bit row format and of windowed attention, in 64 bits (numpy).

TEST INFRASTRUCTURE -- see ``oracle/__init__.py``.

The reference has neither: its caches keep the model's dtype (``pace/llm/cache.py:255-266``) and its attention reads every
cached token its mask allows (``csrc/ops/kernels/attention_kernels.cpp:218-257``).  The format is stated in
``include/pace_kv_hip.h``; a row read back is the bf16 nearest to what its codes stand for.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np
import torch

GROUP = 32
CLAMP = 32768.0


def quantise(x: torch.Tensor) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Codes (int8), steps and middles (float16) of rows ``[..., D]``."""
    y = x.detach().cpu().double().numpy()
    y = np.where(np.isnan(y), 0.0, np.clip(y, -CLAMP, CLAMP))
    y = y.reshape(*y.shape[:-1], y.shape[-1] // GROUP, GROUP)
    lo, hi = y.min(-1), y.max(-1)
    width = hi - lo
    s = (width / 15.0).astype(np.float16)
    s = np.where(15.0 * s.astype(np.float64) < width, np.nextafter(s, np.float16(np.inf)), s)
    below = np.where(s > 0, np.nextafter(s, np.float16(0)), s)
    s = np.where((s > 0) & (15.0 * below.astype(np.float64) >= width), below, s)
    m = (lo + 8.0 * s.astype(np.float64)).astype(np.float32).astype(np.float16)
    step = np.where(s > 0, s.astype(np.float64), 1.0)[..., None]
    code = np.clip(np.rint((y - m.astype(np.float64)[..., None]) / step), -8, 7)
    return np.where(s[..., None] > 0, code, 0).astype(np.int8), s, m


def values64(x: torch.Tensor) -> torch.Tensor:
    """What the stored form of ``x [..., D]`` stands for, in float64."""
    code, s, m = quantise(x)
    v = code.astype(np.float64) * s.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]
    return torch.from_numpy(v.reshape(tuple(x.shape)))


def values_bf16(x: torch.Tensor) -> torch.Tensor:
    """What a gather returns for rows ``x``: the value in single precision, rounded to bf16."""
    return values64(x).float().bfloat16()


def readable(n: int, rows: int, window: int = 0, sinks: int = 0, start: int = 0, causal: bool = True) -> torch.Tensor:
    """``[rows, n]`` bool: which tokens the last ``rows`` positions of a sequence of ``n`` read."""
    pos = (n - rows + torch.arange(rows))[:, None]
    t = torch.arange(n)[None]
    ok = (t >= start).expand(rows, n).clone()
    if causal:
        ok &= t <= pos
    if window:
        ok &= (t > pos - window) | (t < start + sinks)
    return ok


def attention64(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ok: torch.Tensor, mask: Optional[torch.Tensor] = None):
    """One sequence: ``q [Hq, S, D]``, ``k`` / ``v [H, n, D]``, ``ok [S, n]``, additive ``mask [S, n]``.

    Returns the output and what rounding errors are amplified by (for ``error_bound``): the weighted sum of ``|v|``, the largest
    ``scale * sum |q k|`` of a row, and the plain sum of ``|v|`` over the tokens a row reads; all float64.  Rows that read nothing are zero.  Mask values are held at -2^100, so a row
    masked in every column is the average of the tokens it may read.
    """
    hq, S, D = q.shape
    H, n, _ = k.shape
    rep = hq // H
    q, k, v = q.double(), k.double().repeat_interleave(rep, 0), v.double().repeat_interleave(rep, 0)
    scale = 1.0 / math.sqrt(D)
    v = torch.where(ok.any(0)[None, :, None], v, 0.0)  # what no row reads may hold anything
    k = torch.where(ok.any(0)[None, :, None], k, 0.0)
    s = torch.einsum("hsd,hnd->hsn", q, k) * scale
    amp = torch.einsum("hsd,hnd->hsn", q.abs(), k.abs()) * scale
    amp = torch.where(ok[None], amp, 0.0)
    if mask is not None:
        m = mask.double()
        s = torch.where(m[None] <= -(2.0 ** 100), torch.full_like(s, -(2.0 ** 100)), s + m[None])
    s = s.masked_fill(~ok[None], -math.inf)
    top = s.amax(-1, keepdim=True) if n else s.new_zeros(hq, S, 1)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    return p @ v, (p @ v.abs(), amp.amax(-1, keepdim=True) if n else s.new_zeros(hq, S, 1), ok.double()[None] @ v.abs())


def error_bound(out: torch.Tensor, amplified, bits: int) -> torch.Tensor:
    """Elementwise bound of the kernels' error, from the roundings they make (half a step each, ``finfo.eps / 2``):

    * the output to bf16: 2^-8 |out|;
    * 4-bit pools: K, V and the weights to halves, 2^-11 each.  K moves a score by up to 2^-11 * amp, which moves every
      weight by that factor and the sum of the weights by as much again;
    * 4-bit pools, weights under a half's normal range: the row's largest weight is 2^7 or more on the kernels' scale, a half
      below 2^-14 is off by up to 2^-25, so relative to the largest weight (and so to the sum, which is no less) such a
      weight is off by up to 2^-32, whatever its size: 2^-32 times the plain sum of |v|;
    * 16-bit pools: the weights to bf16, 2^-8 (K and V are exact);
    * single-precision sums, the hardware exponential and the score's own rounding: 2^-24 * (256 terms and 2 amp log2 e) and
      2^-20, taken together as 2^-14 (1 + amp).
    """
    spread, amp, reach = amplified
    operand = 2.0 ** -11 * (2 + 2 * amp) if bits == 4 else torch.full_like(amp, 2.0 ** -8)
    return 2.0 ** -8 * out.abs() + spread * (operand * 1.05 + 2.0 ** -14 * (1 + amp)) + (2.0 ** -32 * reach if bits == 4 else 0) + 1e-30
