"""8-bit products for training beside the optimizer: e4m3 codes with a fp32 scale for each block of 128.

``Dion`` steps fp32 master weights; the forward and backward passes between two steps may run in
fewer bits.  ``quantize_rows`` gives activations and gradients a scale for each 1 x 128 block,
``quantize_tiles`` weights one for each 128 x 128 tile, ``float8_product`` multiplies two such
matrices on the tensor cores with fp32 sums, and ``Float8Linear`` is a linear layer made of the
three: forward, gradient of the input, and the gradient of the weight in fp32, as the step takes it.

There is no counterpart in the reference.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Any

import torch
from torch import Tensor, nn

from dionw_b200 import _native

BLOCK = 128
CODES = torch.float8_e4m3fn
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _padded(n: int) -> int:
    """Leading dimension of a matrix of codes: rows start on 16-byte boundaries."""
    return (n + 15) // 16 * 16


@dataclass(frozen=True, init=False, eq=False)
class Float8Matrix:
    """A ``[rows, cols]`` matrix of e4m3 codes and its fp32 scales.

    ``scales`` is ``[rows, ceil(cols / 128)]``, one for each 1 x 128 block, or
    ``[ceil(rows / 128), ceil(cols / 128)]``, one for each tile; of any strides.  An element is its code
    times its block's scale.  Rows of codes start on 16-byte boundaries, a multiple of 16 bytes apart.

    Raises:
        TypeError: On other dtypes.
        ValueError: On shapes, strides or devices that do not fit.
    """

    values: Tensor
    scales: Tensor

    def __init__(self, values: Tensor, scales: Tensor) -> None:
        if values.dtype is not CODES or scales.dtype is not torch.float32:
            raise TypeError(f"Float8Matrix needs float8_e4m3fn codes and float32 scales, got {values.dtype}, {scales.dtype}")
        if values.ndim != 2 or scales.ndim != 2 or values.device != scales.device:
            raise ValueError(
                f"Float8Matrix needs two matrices on one device, got shapes {tuple(values.shape)} on {values.device} and "
                f"{tuple(scales.shape)} on {scales.device}")
        rows, cols = values.shape
        scale_rows, blocks = scales.shape
        if blocks != (cols + 127) // BLOCK or (scale_rows != rows and scale_rows != (rows + 127) // BLOCK):
            raise ValueError(f"scales {tuple(scales.shape)} fit neither the rows nor the tiles of {tuple(values.shape)} codes")
        ld, step = values.stride()
        if ((cols > 1 and step != 1) or values.data_ptr() & 15 or (rows > 1 and (ld & 15 or ld < cols))) and rows and cols:
            raise ValueError(f"rows of codes must start on 16-byte boundaries, got strides {values.stride()}")
        fields = self.__dict__   # (a frozen dataclass's own way costs a microsecond)
        fields["values"], fields["scales"] = values, scales

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def tiles(self) -> bool:
        """Whether 128 rows share a scale."""
        return self.scales.shape[0] != self.values.shape[0]

    def dequantize(self) -> Tensor:
        """The fp32 matrix."""
        rows, cols = self.values.shape
        scales = self.scales.repeat_interleave(BLOCK, 0)[:rows] if self.tiles else self.scales
        return self.values.float() * scales.repeat_interleave(BLOCK, 1)[:, :cols]


def _room(rows: int, cols: int, tiles: bool, device: torch.device) -> tuple[Float8Matrix, tuple[int, int, int, int]]:
    """A matrix to quantize into, and how the quantizer is told of it: codes, their leading dimension, scales, theirs."""
    ld, blocks = (cols + 15) // 16 * 16, (cols + BLOCK - 1) // BLOCK
    values = torch.empty(rows, ld, dtype=CODES, device=device)
    if tiles:
        scales, lds = torch.empty(_blocks(rows), blocks, dtype=torch.float32, device=device), blocks
    else:   # of single rows: those of a block together, as the product and the quantizer go through them
        scales, lds = torch.empty_strided((rows, blocks), (1, rows), dtype=torch.float32, device=device), rows
    target = values.data_ptr(), ld, scales.data_ptr(), lds
    matrix = object.__new__(Float8Matrix)   # nothing to check
    matrix.__dict__.update(values=values if ld == cols else values[:, :cols], scales=scales)
    return matrix, target


def _require_source(x: Tensor) -> None:
    if x.ndim != 2:
        raise ValueError(f"expected a matrix, got shape {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"dionw_b200 quantizes on CUDA devices only, got a matrix on {x.device}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"dionw_b200 quantizes float32, float16 and bfloat16, got {x.dtype}")


def _with_rows(x: Tensor) -> tuple[Tensor, int]:
    """``x``, or a copy, with contiguous rows that do not overlap, and its leading dimension."""
    rows, cols = x.shape
    if cols > 1 and x.stride(1) != 1:
        return x.contiguous(), cols
    ld = x.stride(0)
    if rows > 1 and ld < cols:
        return x.contiguous(), cols
    return x, ld if rows > 1 else cols


_NOWHERE = (None, 0, None, 0)


def _quantize(x: Tensor, tiles: bool, transposed: bool) -> Any:
    _require_source(x)
    x, ldx = _with_rows(x)
    (rows, cols), device = x.shape, x.device
    matrix, target = _room(rows, cols, tiles, device)
    turned, target_t = _room(cols, rows, tiles, device) if transposed else (None, _NOWHERE)
    if rows and cols:
        _native.float8_quantize(x.get_device(), x.data_ptr(), x.dtype, rows, cols, ldx, tiles, *target, *target_t)
    return (matrix, turned) if transposed else matrix


def quantize_rows(x: Tensor, *, transposed: bool = False) -> Any:
    """``x`` ``[rows, cols]`` with a scale for each 1 x 128 block of its rows.

    Codes are rounded to nearest even; a scale is the least power of two that keeps its block in range.
    With ``transposed=True`` returns a pair: the matrix and its transpose (scales along ``x``'s columns),
    from one read.  No gradient passes through (``float8_linear`` has its own).

    Raises:
        ValueError: If ``x`` is not a CUDA matrix.
        TypeError: If it is not float32, float16 or bfloat16.
    """
    return _quantize(x, False, transposed)


def quantize_tiles(x: Tensor, *, transposed: bool = False) -> Any:
    """``quantize_rows`` with a scale for each 128 x 128 tile; the transpose has the same codes and scales."""
    return _quantize(x, True, transposed)


def float8_product(a: Float8Matrix, b: Float8Matrix, *, bias: Tensor | None = None, out: Tensor | None = None,
                   accumulate: bool = False, out_dtype: torch.dtype | None = None) -> Tensor:
    """``a @ b.T`` (``a`` ``[m, k]``, ``b`` ``[n, k]``), plus ``bias`` ``[n]``, summed in fp32 and rounded once.

    Scales may have any value, as long as products of a row's and a column's stay within fp32's range; powers of two, as
    the quantizers make them, are the fast ones for large products (the tensor cores apply them).  The same call gives the
    same bits on the same kind of device.

    Args:
        out: ``[m, n]`` result (float32, float16 or bfloat16), rows contiguous; made if None.  Must not overlap
            ``a``, ``b`` or ``bias``.
        accumulate: Add to what ``out`` holds.
        out_dtype: Of the result that is made (bfloat16 if None); must be ``out``'s where both are given.

    Raises:
        ValueError: On shapes, strides or devices that do not fit, or ``accumulate`` without ``out``.
        TypeError: On other dtypes.
    """
    left, right = a.values, b.values
    (m, k), (n, other) = left.shape, right.shape
    number = left.get_device()
    if k != other:
        raise ValueError(f"float8_product: {tuple(a.shape)} and {tuple(b.shape)} differ in their columns")
    if not left.is_cuda or right.get_device() != number:
        raise ValueError(f"float8_product needs operands on one CUDA device, got {left.device} and {right.device}")
    device = left.device
    if out is None:
        if accumulate:
            raise ValueError("float8_product: accumulate needs out")
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        if out_dtype not in _DTYPES:
            raise TypeError(f"float8_product gives float32, float16 or bfloat16, not {out_dtype}")
        out, ldo = torch.empty(m, n, dtype=out_dtype, device=device), n
    else:
        if out.dtype not in _DTYPES or (out_dtype is not None and out_dtype is not out.dtype):
            raise TypeError(f"float8_product: out is {out.dtype}, out_dtype {out_dtype}")
        if out.shape != (m, n) or out.get_device() != number or (m and n and ((n > 1 and out.stride(1) != 1)
                                                                              or (m > 1 and out.stride(0) < n))):
            raise ValueError(f"float8_product: out must be a [{m}, {n}] matrix with contiguous rows on {device}, "
                             f"got {tuple(out.shape)} with strides {out.stride()} on {out.device}")
        ldo = out.stride(0) if m > 1 else n
    if bias is not None:
        if bias.dtype not in _DTYPES:
            raise TypeError(f"float8_product: bias is {bias.dtype}")
        if bias.shape != (n,) or bias.device != device:
            raise ValueError(f"float8_product: bias must have {n} elements on {device}, got {tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
    if m and n:
        scratch = _product_scratch(number, m, n, k)
        _native.float8_product(number, _operand(left, a.scales, m, k), _operand(right, b.scales, n, k), bias, out, ldo, accumulate,
                               m, n, k, torch.empty(scratch, dtype=torch.uint8, device=device) if scratch else None)
    return out


@functools.lru_cache(maxsize=256)
def _product_scratch(device: int, m: int, n: int, k: int) -> int:
    return _native.float8_product_workspace_bytes(device, m, n, k)


def _operand(values: Tensor, scales: Tensor, rows: int, cols: int) -> tuple[int, int, int, int, int, bool]:
    row_stride, block_stride = scales.stride()
    return (values.data_ptr(), values.stride(0) if rows > 1 else _padded(cols), scales.data_ptr(), row_stride, block_stride,
            scales.shape[0] != rows)


@functools.lru_cache(maxsize=256)
def _packed_bytes(rows: int, cols: int, tiles: bool) -> int:
    return _native.float8_packed_bytes(rows, cols, tiles)


def _kept_at(kept: Tensor | None, x_bytes: int, need_x: bool, need_w: bool) -> tuple[int | None, int | None]:
    """Addresses of the packed transposes of a layer's input and weight."""
    if kept is None:
        return None, None
    at = kept.data_ptr()
    return at if need_w else None, at + x_bytes if need_x else None


class _Linear(torch.autograd.Function):
    """``x @ weight.T`` on 8-bit products; every operand is quantized along the side that is summed over.

    A pass is one call into the library: a layer's host time is most of what small ones take.
    """

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None, recorded: bool) -> Tensor:
        # needs_input_grad says which inputs require gradients; that none is wanted of this call, only its caller knows
        need_x, need_w = (need and recorded for need in ctx.needs_input_grad[:2])
        (tokens, inputs), outputs, device = x.shape, weight.shape[0], x.device
        x_rows, ldx = _with_rows(x)
        w_rows, ldw = _with_rows(weight)
        # What the backward pass needs, a byte an element: the packed transposes of both, x's first.
        x_bytes = _packed_bytes(inputs, tokens, False) if need_w else 0
        kept_bytes = x_bytes + (_packed_bytes(inputs, outputs, True) if need_x else 0)
        kept = torch.empty(kept_bytes, dtype=torch.uint8, device=device) if kept_bytes else None
        x_kept, w_kept = _kept_at(kept, x_bytes, need_x, need_w)
        work = torch.empty(_packed_bytes(tokens, inputs, False) + _packed_bytes(outputs, inputs, True), dtype=torch.uint8,
                           device=device)
        y = torch.empty(tokens, outputs, dtype=x.dtype, device=device)
        _native.float8_linear_forward(x_rows, ldx, w_rows, ldw, None if bias is None else bias.contiguous(), y, tokens, inputs,
                                      outputs, work, x_kept, w_kept)
        ctx.save_for_backward(kept)
        ctx.made_of = (tokens, inputs, outputs, x.dtype, weight.dtype, None if bias is None else bias.dtype, x_bytes)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad: Tensor) -> tuple[Tensor | None, ...]:
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        tokens, inputs, outputs, x_dtype, w_dtype, b_dtype, x_bytes = ctx.made_of
        kept, = ctx.saved_tensors
        x_kept, w_kept = _kept_at(kept, x_bytes, need_x, need_w)
        device = grad.device
        dx = torch.empty(tokens, inputs, dtype=x_dtype, device=device) if need_x else None
        dw = torch.empty(outputs, inputs, dtype=w_dtype, device=device) if need_w else None
        db = torch.empty(outputs, dtype=torch.float32, device=device) if need_b else None
        work = torch.empty((_packed_bytes(tokens, outputs, False) if need_x else 0)
                           + (_packed_bytes(outputs, tokens, False) if need_w else 0), dtype=torch.uint8, device=device)
        dy, ldy = _with_rows(grad)
        _native.float8_linear_backward(dy, ldy, dx, dw, db, tokens, inputs, outputs, work, x_kept, w_kept)
        return dx, dw, db if db is None or b_dtype is torch.float32 else db.to(b_dtype), None


def float8_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """``torch.nn.functional.linear`` with its three products in 8 bits.

    ``x`` is ``[..., inputs]``, ``weight`` ``[outputs, inputs]`` (an fp32 master weight, or 2 bytes), the result has
    ``x``'s dtype, and the weight's gradient the weight's.  Activations and output gradients get a scale for each 1 x 128
    block along the side that is summed over, the weight one for each 128 x 128 tile.  A pass without gradients keeps
    nothing.  Both passes may be captured into a CUDA graph; as with any layer, let no graph of an eager call on the same
    leaves live on meanwhile.  Second derivatives, forward-mode derivatives, ``vmap`` and tracing by ``torch.compile`` are
    not supported.

    Raises:
        ValueError: On shapes that do not fit, or tensors off CUDA or on different devices.
        TypeError: If a dtype is not float32, float16 or bfloat16.
    """
    if weight.ndim != 2 or x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"float8_linear: x {tuple(x.shape)} does not fit a weight {tuple(weight.shape)}")
    number = x.get_device()
    for name, t in (("x", x), ("weight", weight)) if bias is None else (("x", x), ("weight", weight), ("bias", bias)):
        if t.dtype not in _DTYPES:
            raise TypeError(f"float8_linear takes float32, float16 and bfloat16, {name} is {t.dtype}")
        if not t.is_cuda or t.get_device() != number:
            raise ValueError(f"float8_linear needs its tensors on one CUDA device, {name} is on {t.device}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"float8_linear: bias {tuple(bias.shape)} does not fit a weight {tuple(weight.shape)}")
    recorded = torch.is_grad_enabled()   # (never so inside a function's forward)
    if x.ndim == 2:
        return _Linear.apply(x, weight, bias, recorded)
    leading = x.shape[:-1]
    return _Linear.apply(x.reshape(math.prod(leading), x.shape[-1]), weight, bias, recorded).view(*leading, weight.shape[0])


class Float8Linear(nn.Linear):
    """``nn.Linear`` on ``float8_linear``: fp32 master weight and bias, the result in the input's dtype.

    ``param_groups`` routes its weight as any linear layer's; under autocast the input is cast first.
    """

    def forward(self, x: Tensor) -> Tensor:
        if torch.is_autocast_enabled("cuda"):
            x = x.to(torch.get_autocast_dtype("cuda"))
        return float8_linear(x, self.weight, self.bias)
