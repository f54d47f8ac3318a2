"""Loading 8-bit AdamW moments: each optimizer has a state of its own, and the load takes no more room than it."""

from __future__ import annotations

import copy

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


def test_loading_takes_the_room_of_the_codes() -> None:
    """Two bytes an element and the scales, beside what the optimizer holds already: no fp32 copies on the way."""
    n = 1 << 24
    optimizer = _optimizer([n, n])
    _step(optimizer, 0)
    saved = copy.deepcopy(optimizer.state_dict())
    for entry in saved["state"].values():
        for key, value in entry.items():
            entry[key] = value.cpu() if isinstance(value, Tensor) else value
    expect = _state(optimizer)
    _step(optimizer, 1)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    optimizer.load_state_dict(saved)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 2 * n * (2 + 8 / 128) + (1 << 20)
    assert _same(_state(optimizer), expect)


def test_loading_hooks_see_the_moments() -> None:
    optimizer = _optimizer([300])
    _step(optimizer, 0)
    saved = copy.deepcopy(optimizer.state_dict())
    expect = _state(optimizer)
    seen = []

    def before(opt: dionw.Dion, loading: dict) -> dict:
        seen.append({key: value.dtype for key, value in loading["state"][0].items()})
        return loading

    def after(opt: dionw.Dion) -> None:
        entry = opt.state[opt.param_groups[0]["params"][0]]
        seen.append({key: entry[key].dtype for key in KEYS})

    fresh = _optimizer([300], seed=1)
    fresh.register_load_state_dict_pre_hook(before)
    fresh.register_load_state_dict_post_hook(after)
    for _ in range(2):   # what one load sets up is gone before the next
        fresh.load_state_dict(saved)
    dtypes = dict(zip(KEYS, (torch.float8_e4m3fn, torch.float8_e5m2, torch.float32, torch.float32, torch.float32)))
    assert seen == [dtypes] * 4
    assert _same(_state(fresh), expect)


def test_a_checkpoint_that_does_not_fit_leaves_the_loader_as_it_was() -> None:
    optimizer = _optimizer([300])
    _step(optimizer, 0)
    saved, expect = copy.deepcopy(optimizer.state_dict()), _state(optimizer)
    broken = {**saved, "param_groups": [{**saved["param_groups"][0], "params": [0, 1]}]}
    with pytest.raises(ValueError):
        optimizer.load_state_dict(broken)
    assert _same(_state(optimizer), expect)
    optimizer.load_state_dict(saved)
    assert _same(_state(optimizer), expect)
