"""The AdamW route: one fused multi-tensor launch per group (src/dionw/_adamw.py:18-61).

A group with ``adamw_state_bits = 8`` keeps its moments as 8-bit codes with block scales (``adamw8.py``)."""

from __future__ import annotations

from array import array
from collections.abc import Callable
from typing import Any

import torch
from torch import Tensor

from dionw_b200 import _native
from dionw_b200._keys import (
    ADAMW_STATE_BITS_KEY, ADAMW_STEP_STATE, EXP_AVG_SCALE_STATE, EXP_AVG_SQ_SCALE_STATE, EXP_AVG_SQ_STATE, EXP_AVG_STATE,
    ParamState,
)
from dionw_b200.adamw8 import adamw8_state, expected_kinds


def init_adamw_state(param: Tensor, state: dict[str, Any], bits: int = 32) -> None:
    """Fresh moments and an fp32 step counter on the parameter's device."""
    if bits == 8:
        state.update(adamw8_state(param))
        return
    state[EXP_AVG_STATE] = torch.zeros_like(param)
    state[EXP_AVG_SQ_STATE] = torch.zeros_like(param)
    state[ADAMW_STEP_STATE] = torch.zeros((), dtype=torch.float32, device=param.device)


def adamw_step(group: dict[str, Any], state: ParamState,
               hyper: Callable[[torch.device], Tensor | None] | None = None) -> None:
    """One decoupled-decay AdamW step for the group's parameters that have gradients.

    ``hyper(device)`` gives the two-element fp32 device tensor ``{lr, weight_decay}`` the kernel reads
    instead of the host values (so a scheduled learning rate changes no launch), or None."""
    params = [p for p in group["params"] if p.grad is not None]
    if not params:
        return
    devices = {p.device for p in params}
    if len(devices) > 1:   # one launch per device, each with that device current
        for device in sorted(devices, key=lambda d: d.index or 0):
            adamw_step({**group, "params": [p for p in params if p.device == device]}, state, hyper)
        return
    device = params[0].device
    bits = group.get(ADAMW_STATE_BITS_KEY, 32)
    fixups: list[tuple[Tensor, Tensor]] = []
    p_list, g_list, m_list, v_list, s_list = [], [], [], [], []
    scales: tuple[list[Tensor], list[Tensor]] = ([], [])
    for param in params:
        entry = state[param]
        if EXP_AVG_STATE not in entry:
            init_adamw_state(param, entry, bits)
        if (EXP_AVG_SCALE_STATE in entry) != (bits == 8):
            raise ValueError(f"a group's {ADAMW_STATE_BITS_KEY} cannot change once its moments exist")
        grad = param.grad
        if grad is None:
            raise RuntimeError("an AdamW update holds a parameter without a gradient")
        if grad.dtype is not torch.float32 or not grad.is_contiguous():
            grad = grad.float().contiguous()
        target = param
        if not param.is_contiguous():
            # The kernel walks flat memory: update a packed copy and write it back.
            target = param.detach().contiguous()
            fixups.append((param, target))
        p_list.append(target)
        g_list.append(grad)
        m_list.append(entry[EXP_AVG_STATE])
        v_list.append(entry[EXP_AVG_SQ_STATE])
        s_list.append(entry[ADAMW_STEP_STATE])
        if bits == 8:
            scales[0].append(entry[EXP_AVG_SCALE_STATE])
            scales[1].append(entry[EXP_AVG_SQ_SCALE_STATE])
    beta1, beta2 = group["betas"]
    settings = dict(lr=float(group["lr"]), beta1=float(beta1), beta2=float(beta2),
                    weight_decay=float(group["weight_decay"]), eps=float(group["eps"]),
                    hyper_device=None if hyper is None else hyper(device))
    if bits == 8:
        if device.type != "cuda":
            raise ValueError(f"an AdamW update runs on one CUDA device, not on {device}")
        tensors = [*p_list, *g_list, *m_list, *v_list, *scales[0], *scales[1], *s_list]
        addresses, sizes, kinds = _native.tensor_table(tensors)
        number, n = p_list[0].get_device(), len(p_list)
        if kinds != array("Q", expected_kinds(number, torch.float32, n)):
            raise ValueError(f"an AdamW update needs its parameters, gradients and moments on one CUDA device, not {device} and "
                             f"{sorted({f'{t.dtype} on {t.device}' for t in tensors})}")
        _native.adamw8_multi(addresses, sizes[:n], torch.float32, device=number, seed=0, **settings)
    else:
        with torch.cuda.device(device):
            _native.adamw_multi(p_list, g_list, m_list, v_list, s_list, **settings)
    for param, packed in fixups:
        param.copy_(packed)
