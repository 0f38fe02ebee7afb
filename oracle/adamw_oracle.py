"""TEST INFRASTRUCTURE -- the AdamW step, its 8-bit states and the gradient norm in 64 bits.

Written from the definitions in include/flash_muon_b200.h; nothing in the product imports it.
Everything runs on CPU tensors.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

BLOCK = 32
MASK = 0xffffffff


def adamw(w, g, m, v, t: int, *, lr, betas, eps, weight_decay, scale=1.0):
    """(w, m, v) after step number ``t`` (from 1), all in float64, not rounded."""
    b1, b2 = betas
    w, g, m, v = (x.detach().double().cpu() for x in (w, g, m, v))
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    w = w * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return w, m, v


def mix(x: int) -> int:
    x ^= x >> 16
    x = x * 0xa1c7d3e7 & MASK
    x ^= x >> 15
    x = x * 0x2e3ad36d & MASK
    return x ^ x >> 16


def random_numbers(seed: int, t: int, n: int, start: int = 0) -> tuple[Tensor, Tensor]:
    """The random numbers (0 <= u < 1, multiples of 2^-20) of elements start .. start + n - 1 for the
    first and the second moment."""
    key = mix(mix(seed & MASK) + t & MASK)
    h = [mix((i & MASK) ^ mix(key + (i >> 32) & MASK)) for i in range(start, start + n)]
    return (torch.tensor([x & 0xfffff for x in h], dtype=torch.float64) / 2 ** 20,
            torch.tensor([x >> 12 for x in h], dtype=torch.float64) / 2 ** 20)


def code_values(moment: int) -> Tensor:
    """What the codes 0, 1, ... without a sign stand for at scale 127 (126 and 254 are the last
    numbers)."""
    bias, bits, count = (14, 3, 127) if moment == 1 else (29, 3, 255)
    out = []
    for c in range(count):
        e, f = c >> bits, c & 7
        out.append(f / 8 * 2.0 ** (1 - bias) if e == 0 else (1 + f / 8) * 2.0 ** (e - bias))
    return torch.tensor(out, dtype=torch.float64)


def decode(codes: Tensor, scales: Tensor, moment: int) -> Tensor:
    c = codes.cpu().long()
    unit = torch.ldexp(torch.ones(len(scales), dtype=torch.float64), scales.cpu().long() - 127)
    unit = unit.repeat_interleave(BLOCK)[:len(c)]
    table = code_values(moment)
    if moment == 2:
        return torch.cat([table, torch.tensor([math.inf]).double()])[c] * unit
    x = torch.cat([table, torch.tensor([math.nan]).double()])[c & 127] * unit
    return torch.where(c >= 128, -x, x)


def block_scales(x: Tensor, moment: int) -> Tensor:
    """Exponent bytes of the blocks of ``x`` (float64, a multiple of 32 elements)."""
    mag = torch.where(x.isfinite(), x.abs(), 0.0).view(-1, BLOCK).amax(1)
    _, e = torch.frexp(mag)                        # mag = f * 2^e, 0.5 <= f < 1
    b = torch.where(mag > 0, e.long() + 126, 0)
    return b.clamp(17 if moment == 1 else 32, 253)


def rounding_position(x: Tensor, scales: Tensor, moment: int) -> Tensor:
    """Magnitudes of ``x`` on the axis of the codes: the integer part is the code below, the rest the
    distance to it in steps."""
    y = x.abs() / torch.ldexp(torch.ones(len(scales), dtype=torch.float64), scales.long() - 127).repeat_interleave(BLOCK)
    bias = 14 if moment == 1 else 29
    e = (torch.frexp(y)[1].long() - 1).clamp(min=1 - bias)
    e = torch.where(y > 0, e, 1 - bias)
    k = torch.ldexp(y, 3 - e)                      # 8 .. 16, or below 8 for subnormal codes
    return k + 8 * (e + bias - 1)


def pad(x: Tensor) -> Tensor:
    n = len(x)
    out = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=x.dtype)
    out[:n] = x
    return out


def grad_norm(grads, max_norm=math.inf) -> tuple[float, float]:
    total = math.fsum(float(g.detach().double().cpu().square().sum()) for g in grads)
    norm = math.sqrt(total) if math.isfinite(total) else total
    return norm, (min(1.0, max_norm / (norm + 1e-6)) if math.isfinite(norm) else math.nan)
