"""Loading 8-bit AdamW moments: each optimizer has a state of its own."""

from __future__ import annotations

import pytest
import torch
from torch import Tensor, nn

import dionw_b200 as dionw

pytestmark = pytest.mark.gpu
DEV = "cuda"
KEYS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "adamw_step")


def _optimizer(sizes: list[int], seed: int = 0) -> dionw.Dion:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    params = [nn.Parameter(torch.randn(n, device=DEV, generator=gen)) for n in sizes]
    return dionw.Dion([{"params": params, "dion_route": "adamw"}], lr=1e-3, adamw_state_bits=8)


def _step(optimizer: dionw.Dion, seed: int) -> None:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for p in optimizer.param_groups[0]["params"]:
        p.grad = torch.randn(p.shape, device=DEV, generator=gen)
    optimizer.step()


def _state(optimizer: dionw.Dion) -> list[Tensor]:
    """Copies, codes as bytes."""
    tensors = [optimizer.state[p][key] for p in optimizer.param_groups[0]["params"] for key in KEYS]
    return [(t.view(torch.uint8) if t.element_size() == 1 else t).clone() for t in tensors]


def _same(a: list[Tensor], b: list[Tensor]) -> bool:
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_state_loaded_from_a_living_optimizer_is_a_copy() -> None:
    """Codes without the scales and the step that belong to them are other moments."""
    first, second = _optimizer([300, 5000, 0]), _optimizer([300, 5000, 0])
    for seed in range(2):
        _step(first, seed)
    second.load_state_dict(first.state_dict())
    loaded = _state(first)
    assert _same(_state(second), loaded)
    _step(first, 2)
    assert _same(_state(second), loaded) and not _same(_state(first), loaded)
    # and the loaded one goes on as the other did
    for p, q in zip(first.param_groups[0]["params"], second.param_groups[0]["params"]):
        q.data.copy_(p.data)
    moved = _state(first)
    _step(second, 2)
    assert _same(_state(second), moved) and _same(_state(first), moved)
