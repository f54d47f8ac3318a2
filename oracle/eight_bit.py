"""8-bit AdamW moments, block quantization and 8-bit products in 64 bits, from their definitions (test infrastructure).

Written for the CPU and for reading: every format is the list of its values, rounding looks its neighbours up.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

BLOCK = 128
SMALLEST_SCALE = 2.0**-126


def format_values(mantissa: int, bias: int, count: int) -> Tensor:
    """The values of codes 0 .. count - 1 of an 8-bit format."""
    values = []
    for code in range(count):
        exponent, fraction = code >> mantissa, (code & ((1 << mantissa) - 1)) / (1 << mantissa)
        values.append(fraction * 2.0 ** (1 - bias) if exponent == 0 else (1.0 + fraction) * 2.0 ** (exponent - bias))
    return torch.tensor(values, dtype=torch.float64)


E4M3 = format_values(3, 7, 127)      # up to 448
E5M2 = format_values(2, 15, 124)     # up to 57344


def noise(index: Tensor, step: int, seed: int) -> Tensor:
    """The 32-bit word of element ``index`` (int64)."""
    word = 1 << 32
    key = (step * 0x9E3779B9 + seed) % word
    key = (key ^ (key >> 16)) * 0x85EBCA6B % word
    key ^= key >> 13
    low, high = index % word, index // word
    h = (low * 0x9E3779B1 + key + high * 0xC2B2AE35) % word   # products stay below 2**63 for high < 2**30
    h = ((h ^ (h // 2**16)) * 0x7FEB352D) % word
    return h ^ (h // 2**15)


def stochastic_code(x: Tensor, values: Tensor, noise16: Tensor) -> Tensor:
    """Codes of ``x >= 0``: the one below, or the one above where the share of the way up plus noise / 2^16 reaches 1."""
    below = (torch.searchsorted(values, x, right=True) - 1).clamp(0, len(values) - 2)
    share = (x - values[below]) / (values[below + 1] - values[below])
    return below + torch.floor(share + noise16.double() / 65536.0).clamp(0, 1).long()


def adamw8(p: Tensor, g: Tensor, m: Tensor, v: Tensor, step: int, *, lr: float, betas: tuple[float, float],
           weight_decay: float, eps: float, seed: int) -> dict[str, Tensor]:
    """One step of one flat tensor from its dequantized moments; ``step`` counts this one."""
    beta1, beta2 = betas
    p, g, m, v = (t.double().reshape(-1) for t in (p, g, m, v))
    m = beta1 * m + (1.0 - beta1) * g
    v = beta2 * v + (1.0 - beta2) * g * g
    update = lr / (1.0 - beta1**step) * m / (v.sqrt() / math.sqrt(1.0 - beta2**step) + eps)
    out = {"p": p * (1.0 - lr * weight_decay) - update, "update": update, "m": m, "v": v}
    n = p.numel()
    words = noise(torch.arange(n), step, seed)

    def blocks(t: Tensor) -> Tensor:
        return torch.nn.functional.pad(t, (0, -n % BLOCK)).view(-1, BLOCK)

    for name, moment, values, part in (("m", m, E4M3, words % 65536), ("v", v, E5M2, words // 65536)):
        scale = (blocks(moment.abs()).amax(1) / values[-1]).clamp(min=SMALLEST_SCALE)
        spread = scale.repeat_interleave(BLOCK)[:n]
        code = stochastic_code(moment.abs() / spread, values, part)
        if name == "v":
            code = torch.maximum(code, (moment > 0).long())
        out[f"{name}_scale"], out[f"{name}_value"] = scale, values[code] * moment.sign()
        above, below = (code + 1).clamp(max=len(values) - 1), (code - 1).clamp(min=0)
        out[f"{name}_step"] = torch.maximum(values[above] - values[code], values[code] - values[below]) * spread
    return out


def quantize(x: Tensor, tiles: bool) -> tuple[Tensor, Tensor]:
    """``(values, scales)`` of a matrix: e4m3 to nearest, ties to the even code, times the block's power of two."""
    rows, cols = x.shape
    high = BLOCK if tiles else 1
    values = torch.zeros(rows, cols, dtype=torch.float64)
    scales = torch.zeros(-(-rows // high), -(-cols // BLOCK), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = slice(i * high, (i + 1) * high), slice(j * BLOCK, (j + 1) * BLOCK)
            block = x[at].double()
            largest = float(block.abs().max())
            k = -126
            while largest > 448.0 * 2.0**k:
                k += 1
            scale = 2.0**k if largest > 0.0 else 1.0
            y = block.abs() / scale
            below = (torch.searchsorted(E4M3, y, right=True) - 1).clamp(0, len(E4M3) - 2)
            down, up = y - E4M3[below], E4M3[below + 1] - y
            code = below + ((up < down) | ((up == down) & (below % 2 == 1))).long()
            values[at], scales[i, j] = E4M3[code] * block.sign(), scale
    return values, scales


def spread(values: Tensor, scales: Tensor) -> Tensor:
    """What codes and scales stand for."""
    rows, cols = values.shape
    scales = scales.double()
    if scales.shape[0] != rows:
        scales = scales.repeat_interleave(BLOCK, 0)[:rows]
    return values.double() * scales.repeat_interleave(BLOCK, 1)[:, :cols]
