"""8-bit moments under averages so slow that rounding to nearest would hold them where they are.

Each block of 128 has one element that is at its fixed point, which holds the block's scale, and 127 whose moments
start at a code and have a gradient of 1 from then on: the first moment at 1/4, the second at 1/8, and both go to 1.  A step moves the
first by 0.01 of its distance, at most 0.0075 where half a step of e4m3 is 0.0089, the second by 0.001 of its, at most 0.0009 where half
a step of e5m2 is 0.009: rounded to nearest they never move.  Rounded stochastically their mean is the exact average.

How near the mean of n elements has to be: a code's neighbour is at most x / 4 (e5m2) or x / 8 (e4m3) away, and a step's
rounding has at most the variance (distance moved) x (distance of the codes).  With b the average's factor, c = 1/4 or 1/8 and V the
variance that stays, V <= c (1 - b) (1 + V) / (1 - b^2), so V <= c / (1 + b - c) = 1/7 or 1/15: five standard deviations of the mean are
5 sqrt(V / n).  The noise has 16 bits, so that each step is up to 2^-16 of the codes' distance low: 2^-16 c / (1 - b) in the average.
"""

from __future__ import annotations

import math

import pytest
import torch
from torch import Tensor

import dionw_b200 as dionw
from dionw_b200.adamw8 import dequantize_moments
from oracle import eight_bit as oracle

BETAS = (0.99, 0.999)
STEPS = 1000
HOLDER, START = 16.0, (0.25, 0.125)


def _expected() -> list[float]:
    return [1.0 + (start - 1.0) * beta**STEPS for start, beta in zip(START, BETAS)]


def _tolerance(n: int) -> list[float]:
    return [5.0 * math.sqrt(c / (1.0 + beta - c) / n) + 2.0**-16 * c / (1.0 - beta) for c, beta in zip((1 / 8, 1 / 4), BETAS)]


def _moments(blocks: int) -> tuple[Tensor, Tensor, Tensor]:
    """Gradient and both moments, in 64 bits."""
    g = torch.ones(blocks, 128, dtype=torch.float64)
    m, v = START[0] * g, START[1] * g
    g[:, 0], m[:, 0], v[:, 0] = HOLDER, HOLDER, HOLDER**2
    return g.view(-1), m.view(-1), v.view(-1)


def _means(m: Tensor, v: Tensor) -> list[float]:
    return [float(t.double().view(-1, 128)[:, 1:].mean()) for t in (m, v)]


def _near(means: list[float], n: int) -> list[bool]:
    return [abs(mean - want) <= most for mean, want, most in zip(means, _expected(), _tolerance(n))]


def _by_definition(blocks: int, nearest: bool) -> list[float]:
    g, *moments = _moments(blocks)
    for step in range(1, STEPS + 1):
        words = oracle.noise(torch.arange(g.numel()), step, 0)
        for i, (beta, values, part) in enumerate(zip(BETAS, (oracle.E4M3, oracle.E5M2), (words % 65536, words // 65536))):
            x = beta * moments[i] + (1.0 - beta) * (g if i == 0 else g * g)
            scale = (x.view(-1, 128).amax(1) / values[-1]).repeat_interleave(128)
            # half of the noise's range rounds to nearest
            code = oracle.stochastic_code(x / scale, values, torch.full_like(part, 32768) if nearest else part)
            moments[i] = values[code] * scale
    return _means(*moments)


def test_the_case_tells_stochastic_rounding_from_nearest() -> None:
    blocks = 32
    assert _near(_by_definition(blocks, nearest=False), 127 * blocks) == [True, True]
    stuck = _by_definition(blocks, nearest=True)
    assert _near(stuck, 127 * blocks) == [False, False]
    assert stuck == pytest.approx(START, rel=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[2048 * 128], [32 * 128] * 64])
def test_slow_averages_arrive(sizes) -> None:
    """One tensor, and as many elements in tensors of 4096, which share their noise: as much as one of them says."""
    tensors: dict[str, list[Tensor]] = {key: [] for key in ("p", "g", "m", "v", "ms", "vs", "t")}
    for n in sizes:
        g, m, v = _moments(n // 128)
        scales = HOLDER / 448.0, HOLDER**2 / 57344.0
        values = {"p": torch.zeros(n), "g": g.float(), "m": (m / scales[0]).float().to(torch.float8_e4m3fn),
                  "v": (v / scales[1]).float().to(torch.float8_e5m2), "ms": torch.full((n // 128,), scales[0]),
                  "vs": torch.full((n // 128,), scales[1]), "t": torch.zeros(())}
        for key, value in values.items():
            tensors[key].append(value.cuda())
    for _ in range(STEPS):
        dionw.adamw8_step(tensors["p"], tensors["g"], tensors["m"], tensors["v"], tensors["ms"], tensors["vs"], tensors["t"],
                          lr=1e-3, betas=BETAS)
    for i, n in enumerate(sizes):
        entry = dict(zip(("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"),
                         (tensors[key][i] for key in ("m", "v", "ms", "vs"))))
        means = _means(*dequantize_moments(entry))
        assert _near(means, 127 * n // 128) == [True, True], (means, _expected())
