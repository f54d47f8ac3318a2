"""The operators beside the optimizer step that this package is timed on: 8-bit states and 8-bit products.

Four paths:

* ``adamw8``: one AdamW step over many tensors whose moments are held in 8 bits, in blocks of 128
  consecutive elements with a 32-bit scale each.  Returns weights, moments, scales and step counters.
* ``quantize``: a matrix into e4m3 with a power-of-two scale for each 1 x 128 block of its rows
  (activations, gradients) or each 128 x 128 tile (weights), with the transposed copy or without.
* ``product``: ``A @ B.T`` of two such matrices, with a bias or added to what the result holds.
* ``linear``: a linear layer on those products, forward and both gradients.

Every path has a plain form in elementary operations on 32-bit values, and the package's calls.
"""

from __future__ import annotations

import math
import random
from typing import Any

import torch
from torch import Tensor

own = False

Case = dict[str, Any]
DEVICE = torch.device("cuda", 0)
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128
E4M3_MAX, E5M2_MAX = 448.0, 57344.0
SMALLEST_SCALE = 2.0**-126
HYPER = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "weight_decay": 0.05, "eps": 1e-8}
STEPS_DONE = 1000.0   # a run that is under way

# No drawn case costs more than the largest listed one of its path.
MAX_ADAMW_ELEMENTS = 2 * 128256 * 4096
MAX_QUANTIZE_ELEMENTS = 14336 * 4096
MAX_PRODUCT = (8192, 14336, 14336)
MAX_PRODUCT_FLOPS = 2.0 * 8192 * 14336 * 4096
MAX_LINEAR_FLOPS = 6.0 * 4096 * 4096 * 14336


def _adamw8(name: str, sizes: str, grad: str = "fp32", shift: int = 0) -> Case:
    """``sizes``: element counts, ``24x768`` for 24 tensors of 768; ``shift``: elements that weights and gradients
    start behind a 16-byte boundary."""
    return {"name": name, "path": "adamw8", "sizes": sizes, "grad": grad, "shift": shift}


def _quantize(name: str, rows: int, cols: int, dtype: str, block: str, transposed: bool) -> Case:
    return {"name": name, "path": "quantize", "rows": rows, "cols": cols, "dtype": dtype, "block": block,
            "transposed": transposed}


def _product(name: str, m: int, n: int, k: int, b: str, out: str, bias: bool = False, accumulate: bool = False) -> Case:
    """``b``: the right operand's blocks, ``tiles`` or ``rows``."""
    return {"name": name, "path": "product", "m": m, "n": n, "k": k, "b": b, "out": out, "bias": bias,
            "accumulate": accumulate}


def _linear(name: str, tokens: int, inputs: int, outputs: int, dtype: str, bias: bool) -> Case:
    return {"name": name, "path": "linear", "tokens": tokens, "in": inputs, "out": outputs, "dtype": dtype, "bias": bias}


def listed() -> list[Case]:
    return [
        # One bias vector: the smallest step, latency alone.
        _adamw8("adamw8 4096", "4096"),
        # Every AdamW tensor of a small language model: two tables, 50 vectors.
        _adamw8("adamw8 gpt2-small", "38597376,786432,50x768"),
        # Embedding and head of a large one: the largest that a step meets.
        _adamw8("adamw8 2x128256x4096", "525336576,525336576"),
        # No round sizes, 2-byte gradients, tensors that start between 16-byte boundaries.
        _adamw8("adamw8 ragged bf16", "1,127,129,1658481,1000003,2119183", "bf16", 1),
        # One token on its way into a product.
        _quantize("quantize rows 1x4096 bf16", 1, 4096, "bf16", "rows", False),
        # A batch of activations, kept in the other order too for the weight's gradient.
        _quantize("quantize rows 8192x4096 bf16", 8192, 4096, "bf16", "rows", True),
        # A layer's fp32 master weight, in both orders, once a step.
        _quantize("quantize tiles 14336x4096 fp32", 14336, 4096, "fp32", "tiles", True),
        # Generation: one token through a layer.
        _product("product 1x14336x4096", 1, 14336, 4096, "tiles", "bf16"),
        # Forward of a layer over a training batch: the largest.
        _product("product 8192x14336x4096", 8192, 14336, 4096, "tiles", "bf16"),
        # The weight's gradient, added in fp32 to what earlier batches left; no round sizes.
        _product("product 1531x1100x2927 acc", 1531, 1100, 2927, "rows", "fp32", accumulate=True),
        # A layer's forward and backward: a small model's projection with a bias, and a large one's.
        _linear("linear 1000x768x2304 bias", 1000, 768, 2304, "bf16", True),
        _linear("linear 4096x4096x14336", 4096, 4096, 14336, "bf16", False),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
def _spread(rng: random.Random, low: float, high: float) -> float:
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _size(rng: random.Random, low: int, high: int) -> int:
    """A size of the range: often a multiple of 128 or 8, sometimes any whole number."""
    value = _spread(rng, low, high)
    unit = rng.choice((128, 128, 8, 1))
    return int(min(high, max(low, unit * max(1, round(value / unit)))))


def draw(rng: random.Random) -> Case:
    path = rng.choice(("adamw8", "quantize", "product", "product", "linear"))
    if path == "adamw8":
        sizes, room = [], MAX_ADAMW_ELEMENTS
        for _ in range(rng.randint(1, 12)):
            size = min(room, int(_spread(rng, 1, 3e8)))
            if size > 0:
                sizes.append(f"{size}")
                room -= size
        case = _adamw8("", ",".join(sizes), rng.choice(("fp32", "fp32", "bf16", "fp16")), rng.choice((0, 0, 0, 1)))
    elif path == "quantize":
        rows = _size(rng, 1, 16384)
        cols = min(_size(rng, 1, 16384), MAX_QUANTIZE_ELEMENTS // rows)
        case = _quantize("", rows, cols, rng.choice(tuple(DTYPES)), rng.choice(("rows", "rows", "tiles")),
                         rng.random() < 0.5)
    elif path == "product":
        while True:
            m, n, k = _size(rng, 1, MAX_PRODUCT[0]), _size(rng, 16, MAX_PRODUCT[1]), _size(rng, 16, MAX_PRODUCT[2])
            if 2.0 * m * n * k <= MAX_PRODUCT_FLOPS:
                break
        case = _product("", m, n, k, rng.choice(("tiles", "tiles", "rows")), rng.choice(("bf16", "bf16", "fp16", "fp32")),
                        rng.random() < 0.25, rng.random() < 0.25)
    else:
        while True:
            tokens, inputs, outputs = _size(rng, 1, 8192), _size(rng, 16, 14336), _size(rng, 16, 14336)
            if 6.0 * tokens * inputs * outputs <= MAX_LINEAR_FLOPS:
                break
        case = _linear("", tokens, inputs, outputs, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.3)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _numels(case: Case) -> list[int]:
    out: list[int] = []
    for part in case["sizes"].split(","):
        count, _, size = part.rpartition("x")
        out += [int(size)] * int(count or 1)
    return out


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _pieces(buffer: Tensor, starts: list[int], sizes: list[int]) -> list[Tensor]:
    return [buffer[start:start + size] for start, size in zip(starts, sizes)]


def _prepare_adamw8(case: Case, gen: torch.Generator) -> dict[str, Any]:
    """Tensors as views of flat buffers, each from a multiple of 128 elements on; what lies between them is zero."""
    numels = _numels(case)
    blocks = [_ceil(n, BLOCK) for n in numels]
    starts = [BLOCK * sum(blocks[:i]) for i in range(len(blocks))]
    total, shift = BLOCK * sum(blocks), case["shift"]

    def flat(dtype: torch.dtype = torch.float32) -> Tensor:
        return torch.zeros(total + shift, dtype=dtype, device=DEVICE)[shift:]

    p, g = flat(), flat(DTYPES[case["grad"]])
    m, v = flat().to(torch.float8_e4m3fn), flat().to(torch.float8_e5m2)
    sm = torch.empty(total // BLOCK, device=DEVICE).uniform_(0.5e-6, 2e-6, generator=gen)
    sv = torch.empty(total // BLOCK, device=DEVICE).uniform_(0.5e-10, 2e-10, generator=gen)
    # Gradients of one size within a tensor's block, of others elsewhere; every 13th block has none at all.
    size = torch.empty(total // BLOCK, device=DEVICE).uniform_(-3.0, 0.0, generator=gen)
    size = torch.pow(10.0, size) * 1e-2 * (torch.arange(total // BLOCK, device=DEVICE) % 13 != 12)
    for start, n, k in zip(starts, numels, blocks):
        at = slice(start, start + n)
        p[at].normal_(0.0, 0.02, generator=gen)
        noise = torch.empty(n, device=DEVICE).normal_(0.0, 1.0, generator=gen)
        g[at] = noise * size[start // BLOCK:start // BLOCK + k].repeat_interleave(BLOCK)[:n]
        m[at] = noise.normal_(0.0, 100.0, generator=gen).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        v[at] = noise.normal_(0.0, 100.0, generator=gen).square_().clamp_(0.0, E5M2_MAX).to(torch.float8_e5m2)
    steps = torch.full((len(numels),), STEPS_DONE, device=DEVICE)
    scale_starts = [s // BLOCK for s in starts]
    return {"seed": 17, "numels": numels, "p": p, "g": g, "m": m, "v": v, "sm": sm, "sv": sv, "steps": steps,
            "tensors": [_pieces(x, starts, numels) for x in (p, g, m, v)],
            "scales": [_pieces(x, scale_starts, blocks) for x in (sm, sv)],
            "counters": [steps[i] for i in range(len(numels))]}


def _activations(rows: int, cols: int, dtype: str, gen: torch.Generator) -> Tensor:
    """Values as a layer hands them on: some columns ten and more times the others."""
    x = torch.empty(rows, cols, device=DEVICE).normal_(0.0, 1.0, generator=gen)
    x *= torch.exp(torch.empty(cols, device=DEVICE).normal_(0.0, 0.7, generator=gen))
    return x.to(DTYPES[dtype])


def _padded(values: Tensor) -> Tensor:
    """The same values with rows that start on 16-byte boundaries."""
    rows, cols = values.shape
    out = torch.zeros(rows, _ceil(cols, 16) * 16, dtype=values.dtype, device=values.device)
    out[:, :cols] = values
    return out[:, :cols]


def prepare(case: Case, seed: int) -> dict[str, Any]:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state: dict[str, Any] = {"case": dict(case)}
    if case["path"] == "adamw8":
        return state | _prepare_adamw8(case, gen)
    if case["path"] == "quantize":
        x = _activations(case["rows"], case["cols"], case["dtype"], gen)
        if case["block"] == "tiles":
            x.mul_(0.02)
        return state | {"x": x}
    if case["path"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        for name, rows, block in (("a", m, "rows"), ("b", n, case["b"])):
            values, scales = _plain_quantize(_activations(rows, k, "fp32", gen), block)
            state |= {name: _padded(values), f"{name}_scales": scales}
        if case["bias"]:
            state["bias"] = torch.empty(n, device=DEVICE).normal_(0.0, 1.0, generator=gen).to(DTYPES[case["out"]])
        if case["accumulate"]:
            state["out"] = torch.empty(m, n, device=DEVICE).normal_(0.0, math.sqrt(k), generator=gen).to(DTYPES[case["out"]])
        return state
    tokens, inputs, outputs, dtype = case["tokens"], case["in"], case["out"], case["dtype"]
    state["x"] = _activations(tokens, inputs, dtype, gen).requires_grad_()
    state["weight"] = torch.empty(outputs, inputs, device=DEVICE).normal_(0.0, 0.02, generator=gen).requires_grad_()
    state["dy"] = _activations(tokens, outputs, dtype, gen) * 1e-3
    state["bias"] = torch.empty(outputs, device=DEVICE).normal_(0.0, 0.02, generator=gen).requires_grad_() if case["bias"] else None
    return state


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
_LOW = 0xFFFFFFFF


def _words(numels: list[int], steps: Tensor, seed: int) -> Tensor:
    """A 32-bit word for each element of the flat buffers, from its index in its tensor, the step and the seed."""
    sizes = torch.tensor([_ceil(n, BLOCK) * BLOCK for n in numels], device=DEVICE)
    total = sum(_ceil(n, BLOCK) * BLOCK for n in numels)
    index = torch.arange(total, device=DEVICE) - (sizes.cumsum(0) - sizes).repeat_interleave(sizes, output_size=total)
    key = (steps.to(torch.int64) * 0x9E3779B9 + seed) & _LOW
    key = ((key ^ (key >> 16)) * 0x85EBCA6B) & _LOW
    key = (key ^ (key >> 13)).repeat_interleave(sizes, output_size=total)
    key += (index >> 32) * 0xC2B2AE35
    h = ((index & _LOW) * 0x9E3779B1 + key) & _LOW
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & _LOW
    return h ^ (h >> 15)


def _round_up_or_down(x: Tensor, noise: Tensor, mantissa: int, bias: int, most: int) -> Tensor:
    """The 8-bit code of ``x >= 0``: the code below or the one above, the latter where the 16 bits of ``noise`` are
    less than 2^16 times the share of the way up.  Below the smallest normal number the codes are evenly spaced:
    adding that number turns them into the mantissa."""
    drop = 23 - mantissa
    normal = 2.0 ** (1 - bias)
    low = x < normal
    bits = torch.where(low, x + normal, x).view(torch.int32).to(torch.int64) + (noise << (drop - 16))
    first = (127 - bias) << mantissa
    code = (bits >> drop) - first - (low.to(torch.int64) << mantissa)
    return code.clamp(max=most)


def _plain_adamw8(s: dict[str, Any]) -> dict[str, Tensor]:
    lr, beta1, beta2, decay, eps = HYPER.values()
    p, sm, sv, steps = s["p"], s["sm"], s["sv"], s["steps"]
    steps += 1.0
    sizes = torch.tensor([_ceil(n, BLOCK) for n in s["numels"]], device=DEVICE)
    # powers of the betas in 64 bits: 1 - beta^t is a difference of near values in the first steps
    t = steps.double().repeat_interleave(sizes, output_size=sm.numel())[:, None]
    rate = (lr / (1.0 - beta1**t)).float()
    root2 = torch.sqrt(1.0 - beta2**t).float()
    words = _words(s["numels"], steps, s["seed"]).view(-1, BLOCK)
    g = s["g"].float().view(-1, BLOCK)
    m = beta1 * (s["m"].float().view(-1, BLOCK) * sm[:, None]) + (1.0 - beta1) * g
    v = beta2 * (s["v"].float().view(-1, BLOCK) * sv[:, None]) + (1.0 - beta2) * (g * g)
    w = p.view(-1, BLOCK)
    w = w - (lr * decay) * w
    p.copy_((w - rate * (m / (torch.sqrt(v) / root2 + eps))).view(-1))
    sm.copy_((m.abs().amax(1) / E4M3_MAX).clamp(min=SMALLEST_SCALE))
    sv.copy_((v.amax(1) / E5M2_MAX).clamp(min=SMALLEST_SCALE))
    code = _round_up_or_down(m.abs() * (1.0 / sm)[:, None], words & 0xFFFF, 3, 7, 0x7E)
    code |= (m < 0).to(torch.int64) << 7
    s["m"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    code = _round_up_or_down(v * (1.0 / sv)[:, None], words >> 16, 2, 15, 0x7B)
    code = torch.maximum(code, (v > 0).to(torch.int64))   # a second moment is zero only if it is zero
    s["v"].copy_(code.to(torch.uint8).view(torch.float8_e5m2).view(-1))
    return {name: s[name] for name in ("p", "m", "v", "sm", "sv", "steps")}


def _plain_quantize(x: Tensor, block: str) -> tuple[Tensor, Tensor]:
    """``(values, scales)``: the scale is the least power of two with which the block's largest value fits e4m3."""
    rows, cols = x.shape
    high = BLOCK if block == "tiles" else 1
    x = x.float()
    full = torch.zeros(_ceil(rows, high) * high, _ceil(cols, BLOCK) * BLOCK, device=x.device)
    full[:rows, :cols] = x
    full = full.view(-1, high, full.shape[1] // BLOCK, BLOCK)
    largest = full.abs().amax((1, 3))
    fraction, exponent = torch.frexp(largest)   # 448 = 0.875 * 2^9
    exponent = (exponent.to(torch.int32) - 9 + (fraction > 0.875).to(torch.int32)).clamp(min=-126)
    scales = torch.where(largest > 0, ((exponent + 127) << 23).view(torch.float32), 1.0)
    values = (full / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    return values.reshape(values.shape[0] * high, -1)[:rows, :cols], scales


def _spread_scales(values: Tensor, scales: Tensor) -> Tensor:
    """The values an operand stands for, in 32 bits."""
    rows, cols = values.shape
    if scales.shape[0] != rows:
        scales = scales.repeat_interleave(BLOCK, 0)[:rows]
    return values.float() * scales.repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_linear(s: dict[str, Any]) -> tuple[Tensor | None, ...]:
    x, weight, dy, bias = s["x"], s["weight"], s["dy"], s["bias"]
    forward = _spread_scales(*_plain_quantize(x, "rows")) @ _spread_scales(*_plain_quantize(weight, "tiles")).T
    y = (forward if bias is None else forward + bias).to(x.dtype)
    dx = (_spread_scales(*_plain_quantize(dy, "rows")) @ _spread_scales(*_plain_quantize(weight, "tiles"))).to(x.dtype)
    dw = _spread_scales(*_plain_quantize(dy.T, "rows")) @ _spread_scales(*_plain_quantize(x.T, "rows")).T
    return (y, dx, dw) if bias is None else (y, dx, dw, dy.float().sum(0))


@torch.no_grad()
def _plain(s: dict[str, Any]) -> Any:
    case = s["case"]
    if case["path"] == "adamw8":
        return _plain_adamw8(s)
    if case["path"] == "quantize":
        x, block = s["x"], case["block"]
        found = _plain_quantize(x, block)
        return (*found, *_plain_quantize(x.T, block)) if case["transposed"] else found
    if case["path"] == "product":
        out = _spread_scales(s["a"], s["a_scales"]) @ _spread_scales(s["b"], s["b_scales"]).T
        if case["bias"]:
            out += s["bias"]
        if not case["accumulate"]:
            return out.to(DTYPES[case["out"]])
        s["out"].copy_(out + s["out"])
        return s["out"]
    return _plain_linear(s)


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _package(s: dict[str, Any]) -> Any:
    import dionw_b200 as dionw

    case = s["case"]
    if case["path"] == "adamw8":
        params, grads, exp_avg, exp_avg_sq = s["tensors"]
        scale, scale_sq = s["scales"]
        dionw.adamw8_step(params, grads, exp_avg, exp_avg_sq, scale, scale_sq, s["counters"], lr=HYPER["lr"],
                          betas=(HYPER["beta1"], HYPER["beta2"]), weight_decay=HYPER["weight_decay"], eps=HYPER["eps"],
                          seed=s["seed"])
        return {name: s[name] for name in ("p", "m", "v", "sm", "sv", "steps")}
    if case["path"] == "quantize":
        quantize = dionw.quantize_tiles if case["block"] == "tiles" else dionw.quantize_rows
        if not case["transposed"]:
            q = quantize(s["x"])
            return q.values, q.scales
        q, t = quantize(s["x"], transposed=True)
        return q.values, q.scales, t.values, t.scales
    if case["path"] == "product":
        a = dionw.Float8Matrix(s["a"], s["a_scales"])
        b = dionw.Float8Matrix(s["b"], s["b_scales"])
        return dionw.float8_product(a, b, bias=s.get("bias"), out=s.get("out"), accumulate=case["accumulate"],
                                    out_dtype=DTYPES[case["out"]])
    x, weight, bias = s["x"], s["weight"], s["bias"]
    y = dionw.float8_linear(x, weight, bias)
    leaves = (x, weight) if bias is None else (x, weight, bias)
    return (y, *torch.autograd.grad(y, leaves, s["dy"]))


def run(state: dict[str, Any]) -> Any:
    if own:
        return _package(state)
    return _plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: Case) -> dict[str, float]:
    if case["path"] == "adamw8":
        elements = sum(_numels(case))
        blocks = sum(_ceil(n, BLOCK) for n in _numels(case))
        # weight and both moments read and written, gradient read; scales read and written
        return {"bytes": elements * (12.0 + DTYPES[case["grad"]].itemsize) + 16.0 * blocks, "flops": 20.0 * elements}
    if case["path"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        high = BLOCK if case["block"] == "tiles" else 1
        copies = 1.0 + case["transposed"]
        scales = 4.0 * _ceil(rows, high) * _ceil(cols, BLOCK) + case["transposed"] * 4.0 * _ceil(cols, high) * _ceil(rows, BLOCK)
        return {"bytes": rows * cols * (DTYPES[case["dtype"]].itemsize + copies) + scales, "flops": 2.0 * rows * cols}
    if case["path"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        written = m * n * DTYPES[case["out"]].itemsize * (1.0 + case["accumulate"])
        rows_of_b = _ceil(n, BLOCK) if case["b"] == "tiles" else n
        scales = 4.0 * _ceil(k, BLOCK) * (m + rows_of_b)
        return {"bytes": float(m * k + n * k) + written + scales, "flops": 2.0 * m * n * k}
    tokens, inputs, outputs, size = case["tokens"], case["in"], case["out"], DTYPES[case["dtype"]].itemsize
    # x, weight and the output's gradient read; y, x's and the weight's gradients written
    moved = 2.0 * tokens * (inputs + outputs) * size + 8.0 * inputs * outputs
    return {"bytes": moved, "flops": 6.0 * tokens * inputs * outputs}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------
def _exact_code(x: Tensor, noise: Tensor, mantissa: int, bias: int, most: float) -> Tensor:
    """Stochastic rounding of ``x >= 0`` by its definition, as a value: steps of 2^(exponent - mantissa)."""
    _, exponent = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=1 - bias) - mantissa)
    return (torch.floor(x / step + noise.double() / 65536.0) * step).clamp(max=most)


def _exact_adamw8(case: Case, seed: int) -> dict[str, Tensor]:
    s = prepare(case, seed)
    lr, beta1, beta2, decay, eps = HYPER.values()
    t = STEPS_DONE + 1.0
    out = {name: torch.zeros(s[name].shape, dtype=torch.float64, device=DEVICE) for name in ("p", "m", "v")}
    out |= {name: torch.full_like(s[name], SMALLEST_SCALE, dtype=torch.float64) for name in ("sm", "sv")}
    out["steps"] = s["steps"].double() + 1.0
    start = 0
    for i, n in enumerate(s["numels"]):
        blocks = _ceil(n, BLOCK)
        for first in range(0, blocks, 1 << 20):   # a hundred million elements at a time
            count = min(1 << 20, blocks - first)
            at = slice((start + first) * BLOCK, (start + first + count) * BLOCK)
            row = slice(start + first, start + first + count)
            index = torch.arange(first * BLOCK, (first + count) * BLOCK, device=DEVICE)
            key = (int(t) * 0x9E3779B9 + s["seed"]) % 2**32
            key = (key ^ key >> 16) * 0x85EBCA6B % 2**32
            key ^= key >> 13
            word = (index * 0x9E3779B1 + key).remainder(2**32)   # indices stay below 2^32 here
            word = ((word ^ word // 2**16) * 0x7FEB352D).remainder(2**32)
            word = (word ^ word // 2**15).view(-1, BLOCK)
            p, g, m, v = (s[name][at].double().view(-1, BLOCK) for name in ("p", "g", "m", "v"))
            m = beta1 * m * s["sm"][row].double()[:, None] + (1.0 - beta1) * g
            v = beta2 * v * s["sv"][row].double()[:, None] + (1.0 - beta2) * g**2
            denominator = v.sqrt() / math.sqrt(1.0 - beta2**t) + eps
            out["p"][at] = (p * (1.0 - lr * decay) - lr / (1.0 - beta1**t) * m / denominator).view(-1)
            out["sm"][row] = torch.clamp(m.abs().amax(1) / E4M3_MAX, min=SMALLEST_SCALE)
            out["sv"][row] = torch.clamp(v.amax(1) / E5M2_MAX, min=SMALLEST_SCALE)
            code = _exact_code(m.abs() / out["sm"][row][:, None], word.remainder(65536), 3, 7, E4M3_MAX)
            out["m"][at] = (code * m.sign()).view(-1)
            code = _exact_code(v / out["sv"][row][:, None], word // 65536, 2, 15, E5M2_MAX)
            out["v"][at] = torch.where(v > 0, code.clamp(min=2.0**-16), code).view(-1)
        start += blocks
    return out


def _exact_quantize(x: Tensor, block: str) -> tuple[Tensor, Tensor]:
    rows, cols = x.shape
    high = BLOCK if block == "tiles" else 1
    x = torch.nn.functional.pad(x.detach().double(), (0, -cols % BLOCK, 0, -rows % high))
    blocks = x.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, high))      # [rows / high, high, cols / 128, 128]
    largest = blocks.abs().amax((1, 3), keepdim=True)
    fraction, power = torch.frexp(largest / E4M3_MAX)   # an exact power of two has the fraction 0.5
    power = (power - (fraction == 0.5).to(power.dtype)).clamp(min=-126)
    scale = torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), power), 1.0)
    y = blocks / scale
    _, exponent = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (exponent - 1).clamp(min=-6) - 3)
    values = (torch.round(y / step) * step).flatten(2).flatten(0, 1)   # torch.round: halves to even
    return values[:rows, :cols], scale[:, 0, :, 0]


def _exact_values(values: Tensor, scales: Tensor) -> Tensor:
    rows, cols = values.shape
    row = torch.arange(rows, device=DEVICE) // (1 if scales.shape[0] == rows else BLOCK)
    return values.double() * scales.double()[row][:, torch.arange(cols, device=DEVICE) // BLOCK]


@torch.no_grad()
def exact(case: Case, seed: int) -> Any:
    """What ``run`` returns for ``prepare(case, seed)``, in 64 bits."""
    if case["path"] == "adamw8":
        return _exact_adamw8(case, seed)
    s = prepare(case, seed)
    if case["path"] == "quantize":
        found = _exact_quantize(s["x"], case["block"])
        return (*found, *_exact_quantize(s["x"].T, case["block"])) if case["transposed"] else found
    if case["path"] == "product":
        out = _exact_values(s["a"], s["a_scales"]) @ _exact_values(s["b"], s["b_scales"]).T
        if case["bias"]:
            out += s["bias"].double()
        return out + s["out"].double() if case["accumulate"] else out
    x, dy, weight = s["x"], s["dy"], s["weight"]
    w = _exact_values(*_exact_quantize(weight, "tiles"))
    y = _exact_values(*_exact_quantize(x, "rows")) @ w.T
    dx = _exact_values(*_exact_quantize(dy, "rows")) @ w
    dw = _exact_values(*_exact_quantize(dy.T, "rows")) @ _exact_values(*_exact_quantize(x.T, "rows")).T
    if s["bias"] is None:
        return y, dx, dw
    return y + s["bias"].double(), dx, dw, dy.double().sum(0)
