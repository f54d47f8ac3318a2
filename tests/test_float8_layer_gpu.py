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


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_layer_has_the_layers_gradients(reentrant) -> None:
    from torch.utils.checkpoint import checkpoint

    x, layer = _case()
    dy = torch.randn(70, 192, device=DEV).bfloat16()
    found = []
    for run in (layer, lambda t: checkpoint(layer, t, use_reentrant=reentrant)):
        leaf = x.clone().requires_grad_()
        layer.zero_grad()
        y = run(leaf)
        y.backward(dy)
        found.append((y.detach(), leaf.grad, layer.weight.grad, layer.bias.grad))
    assert all(torch.equal(a, b) for a, b in zip(*found))


def test_passes_of_several_batches_add_their_gradients() -> None:
    """Each batch's gradient, added to the one before by autograd: one fp32 rounding each."""
    x, layer = _case(tokens=200)
    dy = torch.randn(200, 192, device=DEV).bfloat16()
    parts = []
    for at in (slice(0, 70), slice(70, 71), slice(71, 200)):
        layer.zero_grad()
        layer(x[at]).backward(dy[at])
        parts.append([p.grad for p in layer.parameters()])
    layer.zero_grad()
    for at in (slice(0, 70), slice(70, 71), slice(71, 200)):
        layer(x[at]).backward(dy[at])
    for i, p in enumerate(layer.parameters()):
        assert torch.equal(p.grad, parts[0][i] + parts[1][i] + parts[2][i])
    # and of one graph twice
    layer.zero_grad()
    y = layer(x)
    y.backward(dy, retain_graph=True)
    once = layer.weight.grad.clone()
    y.backward(dy)
    assert torch.equal(layer.weight.grad, once + once)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_tensors_of_a_device_that_is_not_current() -> None:
    x, layer = _case()
    dy = torch.randn(70, 192, device=DEV).bfloat16()
    other = torch.device("cuda", 1)
    moved = dionw.Float8Linear(256, 192, device=other)
    moved.load_state_dict(layer.state_dict())
    assert torch.cuda.current_device() == 0
    layer(x).backward(dy)
    y = moved(x.to(other))
    y.backward(dy.to(other))
    assert y.device == other and torch.cuda.current_device() == 0
    assert all(torch.equal(p.grad, q.grad.to(DEV)) for p, q in zip(layer.parameters(), moved.parameters()))
