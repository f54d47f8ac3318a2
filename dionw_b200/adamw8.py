"""AdamW with moments held in 8 bits, as one fused step over many tensors.

The moments of a parameter are an e4m3 and an e5m2 tensor of its shape, and a
fp32 scale for every 128 consecutive elements of each: 2.1 bytes per element
where fp32 moments take 8, and 16.1 bytes of memory traffic a step instead of 28.
They are updated in fp32 and rounded stochastically for the next step, by a hash
of the seed, the step and the element's place in its tensor: the same call gives the same
bits.  Tensors of one call, element by element, share their draws.
``Dion(..., adamw_state_bits=8)`` uses it for every AdamW-routed parameter.

The reference keeps its moments in fp32 (src/dionw/_adamw.py:18-61).
"""

from __future__ import annotations

import functools
import math
from array import array
from collections.abc import Sequence
from typing import Any, NoReturn

import torch
from torch import Tensor

from dionw_b200 import _native
from dionw_b200._keys import (
    ADAMW_STEP_STATE, EXP_AVG_SCALE_STATE, EXP_AVG_SQ_SCALE_STATE, EXP_AVG_SQ_STATE, EXP_AVG_STATE,
)

BLOCK = 128                        # consecutive elements that share a scale
MEAN_DTYPE = torch.float8_e4m3fn
SQUARE_DTYPE = torch.float8_e5m2
_GRAD_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def adamw8_state(param: Tensor) -> dict[str, Tensor]:
    """The state before the first step, under the keys a ``Dion`` state entry has."""
    blocks = -(-param.numel() // BLOCK)
    device = param.device
    return {
        EXP_AVG_STATE: torch.zeros(param.shape, dtype=MEAN_DTYPE, device=device),
        EXP_AVG_SQ_STATE: torch.zeros(param.shape, dtype=SQUARE_DTYPE, device=device),
        EXP_AVG_SCALE_STATE: torch.zeros(blocks, dtype=torch.float32, device=device),
        EXP_AVG_SQ_SCALE_STATE: torch.zeros(blocks, dtype=torch.float32, device=device),
        ADAMW_STEP_STATE: torch.zeros((), dtype=torch.float32, device=device),
    }


def dequantize_moments(entry: dict[str, Any]) -> tuple[Tensor, Tensor]:
    """The fp32 moments that a state entry stands for, in the parameter's shape."""
    def values(codes: Tensor, scales: Tensor) -> Tensor:
        return (codes.float().view(-1) * scales.repeat_interleave(BLOCK)[:codes.numel()]).view(codes.shape)

    return (values(entry[EXP_AVG_STATE], entry[EXP_AVG_SCALE_STATE]),
            values(entry[EXP_AVG_SQ_STATE], entry[EXP_AVG_SQ_SCALE_STATE]))


def adamw8_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avg: Sequence[Tensor],
                exp_avg_sq: Sequence[Tensor], exp_avg_scale: Sequence[Tensor], exp_avg_sq_scale: Sequence[Tensor],
                steps: Sequence[Tensor], *, lr: float, betas: tuple[float, float] = (0.9, 0.95),
                weight_decay: float = 0.0, eps: float = 1e-8, seed: int = 0,
                hyper_device: Tensor | None = None) -> None:
    """One decoupled-decay, bias-corrected AdamW step of every parameter, in place.

    Args:
        params: fp32 CUDA tensors of one device, contiguous, each once.  What is written must not overlap.
        grads: Their gradients, of one dtype (float32, float16 or bfloat16), contiguous.
        exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, steps: The state, as ``adamw8_state`` makes
            it.  Every step counter goes up by one.
        lr, betas, weight_decay, eps: As in ``Dion``.
        seed: Of the stochastic rounding, below 2**32.
        hyper_device: Two fp32 on the device, ``{lr, weight_decay}``, read instead of the two arguments.

    A block of 128 elements in which a moment becomes infinite or NaN is NaN from then on.

    Raises:
        ValueError: On lists or tensors that do not fit one another, hyperparameters out of range, or a
            tensor off CUDA or on another device.
        TypeError: On a dtype other than the ones above.
    """
    lists = (grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, steps)
    if any(len(values) != len(params) for values in lists):
        raise ValueError(f"adamw8_step: {len(params)} parameters, {[len(values) for values in lists]} of the others")
    beta1, beta2 = betas
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"adamw8_step: betas must be in [0, 1), got {betas}")
    if not (eps > 0.0 and lr >= 0.0 and weight_decay >= 0.0 and math.isfinite(lr + weight_decay + eps)):
        raise ValueError("adamw8_step: lr and weight_decay must be >= 0 and eps > 0")
    if not 0 <= seed < 1 << 32:
        raise ValueError(f"adamw8_step: seed must be in [0, 2**32), got {seed}")
    if not params:
        return
    device, grad_dtype = params[0].get_device(), grads[0].dtype
    if not params[0].is_cuda:
        raise ValueError(f"adamw8_step runs on CUDA devices, got a parameter on {params[0].device}")
    if grad_dtype not in _GRAD_DTYPES:
        raise TypeError(f"adamw8_step takes float32, float16 or bfloat16 gradients, got {grad_dtype}")
    # Hundreds of tensors a step: one question to all of them.
    n = len(params)
    tensors = [*params, *grads, *exp_avg, *exp_avg_sq, *exp_avg_scale, *exp_avg_sq_scale, *steps]
    addresses, sizes, kinds = _native.tensor_table(tensors)
    if kinds != array("Q", expected_kinds(device, grad_dtype, n)):
        _refuse_kinds(tensors, device, grad_dtype)
    numels = sizes[:n]
    if sizes.tolist()[n:] != numels.tolist() * 3 + [(numel + 127) // BLOCK for numel in numels] * 2 + [1] * n:
        raise ValueError("adamw8_step: gradients, moments or scales do not have the sizes that their parameters need")
    written = addresses[:n] + addresses[2 * n:]
    if len(set(written)) != 6 * n:   # tensors without elements share the address 0
        written = [a for a in written if a]
        if len(set(written)) != len(written):
            raise ValueError("adamw8_step: a parameter, a moment, a scale or a step counter is given twice")
    if hyper_device is not None and (hyper_device.get_device() != device or hyper_device.dtype is not torch.float32
                                     or hyper_device.numel() != 2 or not hyper_device.is_contiguous()):
        raise ValueError("adamw8_step: hyper_device must be two contiguous float32 on the parameters' device")
    _native.adamw8_multi(addresses, numels, grad_dtype, device=device, lr=lr, beta1=beta1, beta2=beta2,
                         weight_decay=weight_decay, eps=eps, seed=seed, hyper_device=hyper_device)


@functools.lru_cache(maxsize=64)
def _kinds(device: int, grad_dtype: torch.dtype) -> tuple[int, ...]:
    return tuple(_native.tensor_kind(t, device) for t in (torch.float32, grad_dtype, MEAN_DTYPE, SQUARE_DTYPE))


def expected_kinds(device: int, grad_dtype: torch.dtype, n: int) -> list[int]:
    """Of parameters, gradients, the two moments, their scales and step counters, n each, as ``_native.tensor_table`` says it."""
    single, gradient, mean, square = _kinds(device, grad_dtype)
    return [single] * n + [gradient] * n + [mean] * n + [square] * n + [single] * (3 * n)


def _refuse_kinds(tensors: list[Tensor], device: int, grad_dtype: torch.dtype) -> NoReturn:
    n = len(tensors) // 7
    dtypes = [torch.float32] * n + [grad_dtype] * n + [MEAN_DTYPE] * n + [SQUARE_DTYPE] * n + [torch.float32] * (3 * n)
    if [t.dtype for t in tensors] != dtypes:
        raise TypeError(
            f"adamw8_step needs float32 parameters, scales and step counters, {grad_dtype} gradients, {MEAN_DTYPE} and "
            f"{SQUARE_DTYPE} moments, got {sorted({str(t.dtype) for t in tensors})}")
    raise ValueError(f"adamw8_step needs contiguous tensors of device {device}")


def require_adamw8_state(param: Tensor, entry: dict[str, Any]) -> None:
    """Raise ValueError if a state entry is not what ``adamw8_state`` makes for ``param``."""
    for key, expected in adamw8_state(param.detach().to("meta")).items():
        found = entry.get(key)
        if not isinstance(found, Tensor) or found.shape != expected.shape or found.dtype is not expected.dtype:
            raise ValueError(
                f"AdamW state of a parameter of shape {tuple(param.shape)} has no 8-bit {key!r} of shape "
                f"{tuple(expected.shape)}: it was saved with other adamw_state_bits")
