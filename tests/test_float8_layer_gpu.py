"""What an 8-bit layer keeps of a forward pass, and the ways in which training calls it."""

from __future__ import annotations

import pytest
import torch
from torch import Tensor

import dionw_b200 as dionw
from dionw_b200 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(tokens: int = 70, inputs: int = 256, outputs: int = 192, seed: int = 0) -> tuple[Tensor, dionw.Float8Linear]:
    torch.manual_seed(seed)
    layer = dionw.Float8Linear(inputs, outputs, device=DEV)
    return torch.randn(tokens, inputs, device=DEV).bfloat16(), layer


def test_a_pass_without_gradients_keeps_nothing(monkeypatch) -> None:
    kept: list[tuple[bool, bool]] = []
    forward = _native.float8_linear_forward

    def spy(*args):
        kept.append((args[-2] is not None, args[-1] is not None))
        return forward(*args)

    monkeypatch.setattr(_native, "float8_linear_forward", spy)
    x, layer = _case()
    leaf = x.clone().requires_grad_()
    with_gradients = layer(leaf)
    layer(x)
    frozen = dionw.float8_linear(leaf, layer.weight.detach(), layer.bias)
    assert kept == [(True, True), (True, False), (False, True)] and frozen.requires_grad
    kept.clear()
    results = []
    for context in (torch.no_grad, torch.inference_mode):
        with context():
            results += [layer(leaf), layer(x)]
    results += [dionw.float8_linear(x, layer.weight.detach(), layer.bias.detach())]
    assert kept == [(False, False)] * 5
    assert all(torch.equal(r, with_gradients) and not r.requires_grad for r in results)
