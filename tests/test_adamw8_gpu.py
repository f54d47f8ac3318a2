"""AdamW with 8-bit moments against its definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch
from torch import Tensor

import dionw_b200 as dionw
from dionw_b200.adamw8 import dequantize_moments
from oracle import eight_bit as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1, eps=1e-8)


def _tensors(sizes: list[int], dtype: torch.dtype = torch.float32, shift: int = 0, seed: int = 0,
             steps: int = 7) -> dict[str, list[Tensor]]:
    gen = torch.Generator().manual_seed(seed)

    def shifted(t: Tensor) -> Tensor:
        room = torch.empty(t.numel() + shift, dtype=t.dtype, device=DEV)
        room[shift:] = t.to(DEV)
        return room[shift:]

    out: dict[str, list[Tensor]] = {key: [] for key in ("p", "g", "m", "v", "ms", "vs", "t")}
    for n in sizes:
        blocks = -(-n // 128)
        size = 10.0 ** (-4 * torch.rand(blocks, generator=gen)).repeat_interleave(128)[:n]
        out["p"].append(shifted(torch.randn(n, generator=gen) * 0.02))
        out["g"].append(shifted((torch.randn(n, generator=gen) * size).to(dtype)))
        out["m"].append((torch.randn(n, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV))
        out["v"].append((torch.rand(n, generator=gen) * 5e4).to(torch.float8_e5m2).to(DEV))
        out["ms"].append((torch.rand(blocks, generator=gen) * 1e-4).to(DEV))
        out["vs"].append((torch.rand(blocks, generator=gen) * 1e-8).to(DEV))
        out["t"].append(torch.full((), float(steps), device=DEV))
    return out


def _shift_codes(t: dict[str, list[Tensor]], key: str, shift: int) -> None:
    for i, codes in enumerate(t[key]):
        room = torch.zeros(codes.numel() + shift, dtype=torch.uint8, device=DEV)
        room[shift:] = codes.view(torch.uint8)
        t[key][i] = room[shift:].view(codes.dtype)


def _moments(t: dict[str, list[Tensor]], i: int) -> tuple[Tensor, Tensor]:
    return dequantize_moments({"exp_avg": t["m"][i], "exp_avg_sq": t["v"][i], "exp_avg_scale": t["ms"][i],
                               "exp_avg_sq_scale": t["vs"][i]})


def _step(t: dict[str, list[Tensor]], **more) -> None:
    dionw.adamw8_step(*(t[key] for key in ("p", "g", "m", "v", "ms", "vs", "t")), **{**HYPER, **more})


def _check(t: dict[str, list[Tensor]], **more) -> None:
    """One step of every tensor against the oracle.

    The weight: two roundings of its own (2^-24 each), and an update of some ten operations in fp32, of which root,
    quotient and the two powers are good to 2^-22: 2^-19 of it in all.  Moments: two products and a sum, 2^-22 of the
    larger term.  A code may be the neighbour of the oracle's where the share of the way up is that near its noise: the
    share's error is at most 2^-20 of the value over a step of at least 2^-4 of it, a chance of 2^-16.
    """
    settings = {**HYPER, "seed": 0, **more}
    expect = []
    for i, p in enumerate(t["p"]):
        m, v = _moments(t, i)
        expect.append(oracle.adamw8(p.cpu(), t["g"][i].cpu(), m.cpu(), v.cpu(), int(t["t"][i]) + 1, **settings))
    _step(t, **more)
    torch.cuda.synchronize()
    for i, want in enumerate(expect):
        p = t["p"][i].cpu().double()
        assert bool(((p - want["p"]).abs() <= 2.0**-22 * want["p"].abs() + 2.0**-19 * want["update"].abs() + 1e-38).all())
        differ = 0
        for codes, scales, name in ((t["m"][i], t["ms"][i], "m"), (t["v"][i], t["vs"][i], "v")):
            assert bool(((scales.cpu().double() - want[f"{name}_scale"]).abs() <= 2.0**-21 * want[f"{name}_scale"]).all())
            got = codes.cpu().double()
            off = got != want[f"{name}_value"]
            differ += int(off.sum())
            value = got * scales.cpu().double().repeat_interleave(128)[:got.numel()]
            # a neighbour at most (the scale's own error aside)
            assert bool(((value - want[name]).abs() <= 1.001 * want[f"{name}_step"]).all())
        n = p.numel()
        assert differ <= 8 + 4 * n * 2.0**-16, differ


@pytest.mark.parametrize("sizes", [[1], [127], [128], [129], [2048], [2049, 1, 4096, 130, 5000], [100_003]])
def test_step_of_sizes(sizes) -> None:
    t = _tensors(sizes)
    _check(t)
    assert all(float(x) == 8.0 for x in t["t"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_step_of_gradient_types_and_alignments(dtype, shift) -> None:
    _check(_tensors([1000, 4096 + 128], dtype, shift, seed=3))


@pytest.mark.parametrize("keys", ["m", "v", "mv"])
@pytest.mark.parametrize("shift", [1, 2, 3, 4])
def test_step_of_codes_between_words(keys, shift) -> None:
    t = _tensors([3000, 129, 1], torch.bfloat16, seed=shift)
    for key in keys:
        _shift_codes(t, key, shift)
    _check(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_elements_give_the_bits_of_a_call_each(dtype) -> None:
    """Whole accesses with more blocks to a warp, from 14.6 M elements on, against tensors between 16-byte boundaries."""
    sizes = [14_600_003, 300, 2048 * 127 + 1, 0, 4096]

    def tensors(shift: int) -> dict[str, list[Tensor]]:
        gen = torch.Generator(device=DEV).manual_seed(3)
        out: dict[str, list[Tensor]] = {key: [] for key in ("p", "g", "m", "v", "ms", "vs", "t")}
        for n in sizes:
            p = torch.empty(n + shift, device=DEV)[shift:].copy_(torch.randn(n, device=DEV, generator=gen) * 0.02)
            g = torch.empty(n + shift, dtype=dtype, device=DEV)[shift:].copy_(torch.randn(n, device=DEV, generator=gen) * 1e-3)
            state = dionw.adamw8_state(p)
            for key, value in zip(out, (p, g, *state.values())):
                out[key].append(value)
        return out

    together, apart = tensors(0), tensors(1)
    for _ in range(3):
        _step(together)
        for i in range(len(sizes)):
            _step({key: values[i:i + 1] for key, values in apart.items()})
    for key in together:
        for a, b in zip(together[key], apart[key]):
            assert torch.equal(a.reshape(-1).view(torch.uint8), b.clone().reshape(-1).view(torch.uint8)), key
    assert [float(t) for t in together["t"]] == [3.0] * len(sizes)
    assert float(together["m"][0].float().abs().max()) == 448.0


def test_what_is_written_twice_is_refused() -> None:
    for key in ("p", "m", "v", "ms", "vs", "t"):
        t = _tensors([256, 256])
        t[key][1] = t[key][0]
        with pytest.raises(ValueError, match="given twice"):
            _step(t)
    t = _tensors([256, 0, 0, 256])
    t["g"][3] = t["g"][0]     # a gradient may serve two
    _check(t)


@pytest.mark.parametrize("more", [
    {"weight_decay": 0.0}, {"betas": (0.0, 0.0)}, {"betas": (0.95, 0.9999)}, {"eps": 1e-3}, {"seed": 2**32 - 1}, {"lr": 0.0}])
def test_step_of_settings(more) -> None:
    _check(_tensors([3000], seed=5), **more)


def test_first_steps_from_the_fresh_state() -> None:
    """The bias corrections of the first steps are differences of near values."""
    t = _tensors([1500], seed=1, steps=0)
    for key in ("m", "v", "ms", "vs"):
        t[key] = [torch.zeros_like(x) for x in t[key]]
    for step in range(3):
        _check(t, betas=(0.9, 0.9999), seed=step)
    fresh = dionw.adamw8_state(t["p"][0].view(3, 500))
    assert fresh["exp_avg"].shape == (3, 500) and fresh["exp_avg_scale"].shape == (12,)


def test_more_tensors_than_a_launch_takes_and_empty_ones() -> None:
    sizes = [0] + [1 + 37 * i for i in range(110)] + [0, 300]
    t = _tensors(sizes, seed=2)
    _check(t)
    assert all(float(x) == 8.0 for x in t["t"])
    only_empty = _tensors([0, 0])
    _step(only_empty)
    assert [float(x) for x in only_empty["t"]] == [8.0, 8.0]


def test_zero_gradients_tiny_and_huge_values() -> None:
    t = _tensors([128 * 6], seed=4)
    g = t["g"][0].view(6, 128)
    g[0] = 0.0                                    # the moments decay
    g[1], t["ms"][0][1], t["vs"][0][1] = 0.0, 0.0, 0.0    # nothing at all: stays zero
    g[2] *= 1e-30 / g[2].abs().max()              # squares below the smallest number
    g[3] = torch.linspace(0, 1e15, 128)
    g[4, 0], g[4, 1:] = 1.0, 1e-12                # one value far above the others
    _check(t)
    assert float(t["m"][0].float().view(6, 128)[1].abs().max()) == 0.0
    # a second moment that is not zero keeps a code that is not zero
    assert float(t["v"][0].float().view(6, 128)[4].min()) > 0.0


def test_infinities_stay_in_their_block() -> None:
    t = _tensors([128 * 4], seed=6)
    t["g"][0].view(4, 128)[1, 5] = math.inf
    t["g"][0].view(4, 128)[3, 7] = math.nan
    before = t["p"][0].clone()
    _step(t)
    assert [bool(x) for x in t["ms"][0].isnan()] == [False, True, False, True]
    assert [bool(x) for x in t["vs"][0].isnan()] == [False, True, False, True]
    bad = ~t["p"][0].isfinite()
    assert bad.nonzero().flatten().tolist() == [128 + 5, 3 * 128 + 7]
    t["g"][0].zero_()
    _step(t)
    assert bool(t["p"][0].view(4, 128)[[1, 3]].isnan().all()) and bool(t["p"][0].view(4, 128)[[0, 2]].isfinite().all())
    assert not bool((t["p"][0] == before).all())


def test_rounding_is_right_on_average_and_moves_slow_averages() -> None:
    """A constant gradient under beta2 = 0.999: the second moment goes up by 0.1 % of its distance each step, far below a
    step of e5m2, and has to arrive all the same.  After 2000 steps the exact one is at 1 - 0.999^2000 = 86.5 % of g^2; the
    codes' noise of 4096 elements averages out: a step's is below a quarter of the value, the average remembers
    1000 of them, of which 0.5 % move, so that the mean is within 4 * 0.25 * sqrt(5) / sqrt(4096) = 4 %."""
    n = 4096
    t = _tensors([n], steps=0)
    t["p"], t["g"] = [torch.zeros(n, device=DEV)], [torch.full((n,), 0.01, device=DEV)]
    for key in ("m", "v", "ms", "vs"):
        t[key] = [torch.zeros_like(x) for x in t[key]]
    # one element of each block is larger, so that the others lie between codes
    t["g"][0].view(-1, 128)[:, 0] = 0.017
    for _ in range(2000):
        _step(t, betas=(0.9, 0.999), weight_decay=0.0)
    _, v = _moments(t, 0)
    inner = v.view(-1, 128)[:, 1:].double()
    assert float(inner.mean()) == pytest.approx(1e-4 * (1 - 0.999**2000), rel=0.04)


def test_same_call_same_bits_and_the_seed_counts() -> None:
    first, second, third = (_tensors([5000, 77], seed=8) for _ in range(3))
    _step(first)
    _step(second)
    _step(third, seed=1)
    for key in first:
        assert all(torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a,
                               b.view(torch.uint8) if b.element_size() == 1 else b) for a, b in zip(first[key], second[key]))
    assert not torch.equal(first["m"][0].view(torch.uint8), third["m"][0].view(torch.uint8))
    assert torch.equal(first["p"][0], third["p"][0])   # the weight moves by what is not rounded


def test_scalars_from_the_device_and_another_stream() -> None:
    first, second = _tensors([3000], seed=9), _tensors([3000], seed=9)
    _step(first, lr=2e-3, weight_decay=0.3)
    table = torch.tensor([2e-3, 0.3], device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(second, lr=5.0, weight_decay=0.0, hyper_device=table)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first["p"][0], second["p"][0])


def test_captured_step_replays() -> None:
    eager, captured = _tensors([3000, 100], seed=10), _tensors([3000, 100], seed=10)
    for _ in range(3):
        _step(eager)
    _step(captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(captured)
    graph.replay()
    graph.replay()
    for key in eager:
        for a, b in zip(eager[key], captured[key]):
            assert torch.equal(a.float(), b.float())
