"""Refusals of the 8-bit entry points; no GPU needed."""

from __future__ import annotations

import contextlib

import pytest
import torch
import torch.distributed as dist

from dionw_b200 import _native
from dionw_b200.distributed import ShardedDion


def test_exponents_of_one_operand_are_refused() -> None:
    """They would go unused, and the product would be summed as one without."""
    lib = _native.library()
    at = 1 << 20   # an address that is never read

    def call(m: int, a_exponents: int | None, b_exponents: int | None) -> int:
        return lib.dionw_float8_product(at, 112, at, 1, m, 0, at, 112, at, 1, 6, 0, None, 0, at, 6, 0, 0, m, 6, 100, a_exponents,
                                        b_exponents, None, 0, None)

    for m in (0, 4, 200):
        for one in ((at, None), (None, at)):
            assert call(m, *one) == -1
            assert "one operand" in _native.last_error()
    assert call(0, at, at) == 0 and call(0, None, None) == 0


def test_sharded_dion_refuses_moments_in_8_bits(tmp_path) -> None:
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        group = {"params": [], "dion_route": "adamw"}
        with pytest.raises(ValueError, match="trainable"):   # 32 is not what is refused
            ShardedDion([{**group, "adamw_state_bits": 32}], lr=1e-3)
        with pytest.raises(NotImplementedError, match="float32"):
            ShardedDion([{**group, "adamw_state_bits": 8}], lr=1e-3)
        with pytest.raises(TypeError, match="adamw_state_bits"):
            ShardedDion([group], lr=1e-3, adamw_state_bits=8)
    finally:
        dist.destroy_process_group()


def test_a_call_runs_on_its_tensors_device(monkeypatch) -> None:
    """The device is made current for the call, where it is not, and the stream is that device's."""
    events: list = []

    @contextlib.contextmanager
    def device(number: int):
        events.append(("enter", number))
        yield
        events.append(("leave", number))

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda number: 1000 + number, raising=False)

    def entry(*args: int) -> int:
        events.append(args)
        return 0

    _native.on_device(1, entry, 5, 6)
    assert events == [(5, 6, 1001)]
    events.clear()
    _native.on_device(3, entry, 5)
    assert events == [("enter", 3), (5, 1003), ("leave", 3)]
