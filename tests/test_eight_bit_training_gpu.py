"""Dion with 8-bit AdamW moments, and a model of 8-bit linear layers trained by it."""

from __future__ import annotations

import copy
import io

import pytest
import torch
from torch import Tensor, nn

import dionw_b200 as dionw
from dionw_b200 import EMAConfig
from dionw_b200.adamw8 import dequantize_moments
from oracle import eight_bit as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Model(nn.Module):
    """A small language model's parts: a table, two 8-bit layers with a norm, a head."""

    def __init__(self, vocab: int = 311, width: int = 192, hidden: int = 320) -> None:
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.up = dionw.Float8Linear(width, hidden)
        self.norm = nn.LayerNorm(hidden)
        self.down = dionw.Float8Linear(hidden, width, bias=False)

    def forward(self, tokens: Tensor) -> Tensor:
        x = self.embed(tokens)
        x = x + self.down(torch.nn.functional.gelu(self.norm(self.up(x.bfloat16()).float())).bfloat16()).float()
        return x @ self.embed.weight.T


def _model(seed: int = 0) -> _Model:
    torch.manual_seed(seed)
    return _Model().to(DEV)


def _optimizer(model: nn.Module, **more) -> dionw.Dion:
    groups, _ = dionw.param_groups(model, min_matrix_dim=8)
    return dionw.Dion(groups, lr=1e-3, weight_decay=0.1, **{"adamw_state_bits": 8, **more})


def _backward(model: nn.Module, seed: int) -> None:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    tokens = torch.randint(0, 311, (3, 70), device=DEV, generator=gen)
    loss = nn.functional.cross_entropy(model(tokens[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())
    model.zero_grad(set_to_none=False)
    loss.backward()


def _codes(t: Tensor) -> Tensor:
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _state(optimizer: dionw.Dion) -> list[Tensor]:
    return [_codes(value) for group in optimizer.param_groups for p in group["params"]
            for _, value in sorted(optimizer.state[p].items()) if isinstance(value, Tensor)]


def test_groups_and_state() -> None:
    model = _model()
    optimizer = _optimizer(model)
    for group in optimizer.param_groups:
        assert group.get("adamw_state_bits") == (8 if group["dion_route"] == "adamw" else None)
    entry = optimizer.state[model.embed.weight]
    assert entry["exp_avg"].dtype is torch.float8_e4m3fn and entry["exp_avg_sq"].dtype is torch.float8_e5m2
    assert entry["exp_avg_scale"].shape == (311 * 192 // 128 + 1,)
    # 32 bits stay what they were, checkpoint keys included
    plain = _optimizer(_model(), adamw_state_bits=32)
    assert all("adamw_state_bits" not in group for group in plain.param_groups)
    groups, _ = dionw.param_groups(_model())
    groups[0]["adamw_state_bits"] = 8
    mixed = dionw.Dion(groups, lr=1e-3)
    assert [g.get("adamw_state_bits") for g in mixed.param_groups][:2] == [8, None]


def test_step_follows_the_definition() -> None:
    model = _model(1)
    optimizer = _optimizer(model)
    for step in range(1, 4):
        _backward(model, step)
        expect = {}
        for group in optimizer.param_groups:
            if group["dion_route"] != "adamw":
                continue
            for p in group["params"]:
                m, v = dequantize_moments(optimizer.state[p])
                expect[p] = oracle.adamw8(p.detach().cpu(), p.grad.cpu(), m.cpu(), v.cpu(), step, lr=group["lr"],
                                          betas=group["betas"], weight_decay=group["weight_decay"], eps=group["eps"], seed=0)
        optimizer.step()
        assert len(expect) == 4   # the table, a bias, the norm's two
        for p, want in expect.items():
            got = p.detach().cpu().double().flatten()
            assert bool(((got - want["p"]).abs() <= 2.0**-22 * want["p"].abs() + 2.0**-19 * want["update"].abs() + 1e-38).all())
            entry = optimizer.state[p]
            for key, name in (("exp_avg", "m"), ("exp_avg_sq", "v")):
                differ = entry[key].cpu().double().flatten() != want[f"{name}_value"]
                assert int(differ.sum()) <= 8 + 4 * got.numel() * 2.0**-16
            assert float(entry["adamw_step"]) == step


def test_checkpoint_resumes_bit_for_bit() -> None:
    model = _model(2)
    optimizer = _optimizer(model, ema=EMAConfig(decay=0.99))
    for step in range(3):
        _backward(model, step)
        optimizer.step()
    file = io.BytesIO()
    torch.save({"model": model.state_dict(), "optimizer": optimizer.state_dict()}, file)
    file.seek(0)
    saved = torch.load(file, weights_only=True)
    other = _model(3)
    resumed = _optimizer(other, ema=EMAConfig(decay=0.99))
    other.load_state_dict(saved["model"])
    resumed.load_state_dict(saved["optimizer"])
    for step in range(3, 6):
        for m, o in ((model, optimizer), (other, resumed)):
            _backward(m, step)
            o.step()
    assert all(torch.equal(a, b) for a, b in zip(model.parameters(), other.parameters()))
    a, b = _state(optimizer), _state(resumed)
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_checkpoint_of_other_bits_is_refused() -> None:
    for bits in (8, 32):
        optimizer = _optimizer(_model(), adamw_state_bits=bits)
        with pytest.raises(ValueError, match="adamw_state_bits"):
            _optimizer(_model(), adamw_state_bits=40 - bits).load_state_dict(optimizer.state_dict())
    optimizer = _optimizer(_model())
    broken = copy.deepcopy(optimizer.state_dict())
    del broken["state"][0]["exp_avg_scale"]
    with pytest.raises(ValueError, match="exp_avg"):
        _optimizer(_model()).load_state_dict(broken)


def test_replayed_steps_are_the_steps() -> None:
    models = [_model(4), _model(4)]
    optimizers = [_optimizer(m) for m in models]
    optimizers[1].graph_replay = True
    for step in range(5):
        for group_a, group_b in zip(optimizers[0].param_groups, optimizers[1].param_groups):
            group_a["lr"] = group_b["lr"] = 1e-3 / (1 + step)
        for m, o in zip(models, optimizers):
            _backward(m, step)
            o.step()
    assert optimizers[1].graph_replays >= 2
    assert all(torch.equal(a, b) for a, b in zip(models[0].parameters(), models[1].parameters()))
    assert all(torch.equal(a, b) for a, b in zip(_state(optimizers[0]), _state(optimizers[1])))


def test_parameters_that_are_not_packed_and_without_gradients() -> None:
    base = torch.randn(40, 30, device=DEV)
    strided = nn.Parameter(base.T)
    packed = nn.Parameter(base.T.contiguous())
    idle = nn.Parameter(torch.randn(7, device=DEV))
    optimizer = dionw.Dion([{"params": [strided, packed, idle], "dion_route": "adamw"}], lr=1e-3, adamw_state_bits=8)
    grad = torch.randn(30, 40, device=DEV)
    strided.grad, packed.grad = grad.T.contiguous().T, grad.clone()
    before = idle.detach().clone()
    optimizer.step()
    assert torch.equal(strided, packed) and torch.equal(idle, before)
    assert float(optimizer.state[idle]["adamw_step"]) == 0.0
    assert torch.equal(_codes(optimizer.state[strided]["exp_avg"]), _codes(optimizer.state[packed]["exp_avg"]))
