"""Block quantization, 8-bit products and the linear layer on them, against their definitions in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch
from torch import Tensor

import dionw_b200 as dionw
from dionw_b200 import Float8Matrix
from oracle import eight_bit as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _matrix(rows: int, cols: int, seed: int = 0, dtype: torch.dtype = torch.float32) -> Tensor:
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen))).to(dtype)


# ---------------------------------------------------------------------------
# quantization: the codes and scales of the definition, bit for bit
# ---------------------------------------------------------------------------
def _same(got: Float8Matrix, x: Tensor, tiles: bool) -> None:
    values, scales = oracle.quantize(x, tiles)
    assert torch.equal(got.values.cpu().double(), values)
    assert torch.equal(got.scales.cpu().double(), scales)


@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 127), (128, 128), (129, 257), (300, 1000), (17, 9)])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize(shape, tiles, dtype) -> None:
    x = _matrix(*shape, dtype=dtype)
    quantize = dionw.quantize_tiles if tiles else dionw.quantize_rows
    _same(quantize(x.to(DEV)), x, tiles)
    straight, transposed = quantize(x.to(DEV), transposed=True)
    _same(straight, x, tiles)
    _same(transposed, x.T, tiles)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_views(dtype) -> None:
    """Rows between 16-byte boundaries, rows apart, columns apart."""
    x = _matrix(200, 301, seed=1, dtype=dtype)
    on = x.to(DEV)
    for view, same in ((on[:, 1:], x[:, 1:]), (on[3:, :160], x[3:, :160]), (on[::2, 5:], x[::2, 5:]), (on.T, x.T),
                       (on[:, ::3], x[:, ::3]), (on[:1, 4:].expand(70, -1), x[:1, 4:].expand(70, -1))):
        straight, transposed = dionw.quantize_rows(view, transposed=True)
        _same(straight, same, False)
        _same(transposed, same.T, False)


def test_quantize_borders() -> None:
    """Largest values at and next to 448 * 2^k, ties between codes, values down to nothing, zeros."""
    x = torch.zeros(12, 256)
    x[0, 0], x[1, 0], x[2, 0] = 448.0, math.nextafter(448.0, 500.0) + 2.0**-15, 447.9
    x[3, :127] = torch.arange(127) * 0.25 - 16.0
    x[4, 0], x[4, 1:20] = 448.0, torch.arange(19) * 2.0**-10          # half steps of the smallest codes
    x[5, 0], x[6, 0], x[7, 0] = 3.4028234e38, 1e-38, 1.4e-45
    x[8, 3], x[9, 128] = -1.0, 1e-20
    x[10, 0], x[10, 1:18] = 16.0 * 28, (16 + torch.arange(17)) / 2 * 1.0
    for tiles in (False, True):
        (dionw.quantize_tiles if tiles else dionw.quantize_rows)(x.to(DEV))
    straight, transposed = dionw.quantize_rows(x.to(DEV), transposed=True)
    _same(straight, x, False)
    _same(transposed, x.T, False)
    _same(dionw.quantize_tiles(x.to(DEV)), x, True)


def test_quantize_infinities_stay_in_their_block() -> None:
    x = _matrix(130, 300, seed=2)
    x[5, 7], x[129, 299], x[40, 200] = math.inf, math.nan, -math.inf
    straight, transposed = dionw.quantize_rows(x.to(DEV), transposed=True)
    assert straight.scales.isnan().nonzero().tolist() == [[5, 0], [40, 1], [129, 2]]
    assert transposed.scales.isnan().nonzero().tolist() == [[7, 0], [200, 0], [299, 1]]
    assert dionw.quantize_tiles(x.to(DEV)).scales.isnan().nonzero().tolist() == [[0, 0], [0, 1], [1, 2]]
    clean = x.clone()
    clean[5, :128], clean[40, 128:256], clean[129, 256:] = 0.0, 0.0, 0.0
    values, _ = oracle.quantize(clean, False)
    keep = clean != 0.0
    assert torch.equal(straight.values.cpu().double()[keep], values[keep])


def test_quantize_leaves_neighbours_alone() -> None:
    """The C entry with room around the codes: only the next multiple of 8 is written."""
    from dionw_b200 import _native

    x = _matrix(70, 133, seed=3).to(DEV)
    q = torch.full((72, 160), 7, dtype=torch.uint8, device=DEV)
    qt = torch.full((140, 96), 7, dtype=torch.uint8, device=DEV)
    scales, scales_t = torch.full((3, 80), 7.0, device=DEV), torch.full((2, 140), 7.0, device=DEV)
    _native.float8_quantize(x.get_device(), x.data_ptr(), x.dtype, 70, 133, 133, False, q.data_ptr(), 160,
                            scales.data_ptr(), 80, qt.data_ptr(), 96, scales_t.data_ptr(), 140)
    assert bool((q[70:] == 7).all()) and bool((q[:, 136:] == 7).all())
    assert bool((qt[133:] == 7).all()) and bool((qt[:, 72:] == 7).all())
    assert bool((scales[2:] == 7).all()) and bool((scales[:, 70:] == 7).all())
    assert bool((scales_t[1:] == 7).all()) and bool((scales_t[:, 133:] == 7).all())


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _operand(rows: int, k: int, tiles: bool, seed: int, layout: str = "blocks") -> tuple[Float8Matrix, Tensor]:
    """Codes of any value, scales that are no powers of two, and the 64-bit matrix; ``layout`` of the scales."""
    gen = torch.Generator().manual_seed(seed)
    room = torch.zeros(rows, (k + 15) // 16 * 16 + 16)
    room[:, :k] = torch.randn(rows, k, generator=gen) * 100
    codes = room.clamp(-448, 448).to(torch.float8_e4m3fn)
    count = -(-rows // 128) if tiles else rows
    scales = torch.exp(torch.randn(count, -(-k // 128), generator=gen)) * 1e-2
    on = scales.to(DEV) if layout == "rows" else scales.T.contiguous().to(DEV).T
    return Float8Matrix(codes.to(DEV)[:, :k], on), oracle.spread(codes[:, :k].float(), scales)


def _close(got: Tensor, a: Tensor, b: Tensor, extra: Tensor | float = 0.0) -> None:
    """Sums of k products in fp32, at most 128 in a row on the tensor cores and then block by block: (32 + blocks)
    roundings of 2^-23 of the sum of the magnitudes, and the rounding of the result."""
    want = a @ b.T + extra
    blocks = -(-a.shape[1] // 128)
    size = a.abs() @ b.abs().T + (extra.abs() if isinstance(extra, Tensor) else 0.0)
    bound = (32 + blocks) * 2.0**-23 * size + HALF_STEP[got.dtype] * 1.01 * want.abs() + 1e-30
    if got.dtype is torch.float16:
        bound = bound + 2.0**-25     # half a step of its smallest numbers
    assert bool(((got.cpu().double() - want).abs() <= bound).all()), float(((got.cpu().double() - want).abs() / bound).max())


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 128), (1, 300, 517), (7, 129, 1000), (16, 256, 384), (17, 1000, 129), (33, 64, 4000), (1, 20000, 300), (5, 130, 14336), (20, 400, 8200), (64, 129, 5000), (2, 1000, 4097),
    (64, 500, 640), (65, 127, 255), (128, 128, 128), (129, 257, 1153), (300, 700, 2048), (256, 256, 8192), (1000, 48, 96)])
@pytest.mark.parametrize("b_tiles", [False, True])
def test_product(m, n, k, b_tiles) -> None:
    a, a64 = _operand(m, k, False, 1)
    b, b64 = _operand(n, k, b_tiles, 2, "rows")
    for dtype in DTYPES:
        _close(dionw.float8_product(a, b, out_dtype=dtype), a64, b64)


@pytest.mark.parametrize("m,n,k", [(2500, 1900, 300), (513, 9500, 1153), (4096, 1280, 127), (2304, 2305, 4100)])
@pytest.mark.parametrize("b_tiles", [False, True])
def test_product_of_many_tiles(m, n, k, b_tiles) -> None:
    """Enough tiles for a pair of SMs each, several for some."""
    a, a64 = _operand(m, k, False, 1)
    b, b64 = _operand(n, k, b_tiles, 2, "rows")
    held = torch.randn(m, n, generator=torch.Generator().manual_seed(3))
    _close(dionw.float8_product(a, b), a64, b64)
    _close(dionw.float8_product(a, b, out=held.to(DEV), accumulate=True), a64, b64, held.double())


@pytest.mark.parametrize("m,n,k", [(2500, 1900, 1153), (513, 9500, 1153), (300, 260, 2400), (1300, 1100, 2900), (200, 4000, 6900)])
@pytest.mark.parametrize("b_tiles", [False, True])
@pytest.mark.parametrize("layout", ["rows", "blocks"])
def test_product_of_many_tiles_and_powers_of_two(m, n, k, b_tiles, layout) -> None:
    """Scales that the tensor cores take; one other one, first or last of either operand, sends the product the other way."""
    from dionw_b200 import _native

    gen = torch.Generator().manual_seed(9)
    (a, _), (b, _) = _operand(m, k, False, 1, layout), _operand(n, k, b_tiles, 2, layout)
    for x in (a, b):
        x.scales.copy_(torch.exp2(torch.randint(-20, 20, x.scales.shape, generator=gen).float()))

    def values(x: Float8Matrix) -> Tensor:
        return oracle.spread(x.values.cpu().float(), x.scales.cpu())

    # (the few tiles of the third one are shared out instead)
    assert (_native.float8_product_workspace_bytes(0, m, n, k) > 0) == (m != 300)
    for dtype in DTYPES[:2]:
        _close(dionw.float8_product(a, b, out_dtype=dtype), values(a), values(b))
    for x, at in ((a, (0, 0)), (a, (-1, -1)), (b, (0, 0)), (b, (-1, -1))):
        for other in (1.5, 0.0, -2.0, 2.0**-130):
            kept = x.scales[at].clone()
            x.scales[at] = other
            _close(dionw.float8_product(a, b), values(a), values(b))
            x.scales[at] = kept
    a.scales[3, 1] = math.nan
    assert dionw.float8_product(a, b).isnan().any(1).nonzero().flatten().tolist() == [3]


@pytest.mark.parametrize("m", [40, 200])
def test_product_with_weights_on_the_left(m) -> None:
    a, a64 = _operand(m, 700, True, 3)
    b, b64 = _operand(150, 700, True, 4)
    _close(dionw.float8_product(a, b, out_dtype=torch.float32), a64, b64)


@pytest.mark.parametrize("m,n", [(3, 200), (200, 333), (130, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_adds_bias_and_what_is_there(m, n, dtype) -> None:
    a, a64 = _operand(m, 300, False, 5)
    b, b64 = _operand(n, 300, True, 6)
    gen = torch.Generator().manual_seed(7)
    bias = (torch.randn(n, generator=gen) * 30).to(dtype)
    held = (torch.randn(m, n, generator=gen) * 30).to(dtype)
    _close(dionw.float8_product(a, b, bias=bias.to(DEV), out_dtype=dtype), a64, b64, bias.double().expand(m, n))
    out = held.to(DEV)
    assert dionw.float8_product(a, b, bias=bias.to(DEV), out=out, accumulate=True) is out
    _close(out, a64, b64, bias.double() + held.double())
    # rows apart, between 16-byte boundaries: neighbours stay as they are
    room = torch.full((m, n + 9), 5.0, dtype=dtype, device=DEV)
    _close(dionw.float8_product(a, b, out=room[:, 3:n + 3]), a64, b64)
    assert bool((room[:, :3] == 5).all()) and bool((room[:, n + 3:] == 5).all())


@pytest.mark.parametrize("m,n,k", [(200, 333, 3001), (66, 1030, 5000), (300, 700, 2048)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_in_parts_adds_bias_and_what_is_there(m, n, k, dtype) -> None:
    """Few tiles with long sums: the CTAs of a cluster share them."""
    a, a64 = _operand(m, k, False, 5, "rows")
    b, b64 = _operand(n, k, False, 6)
    gen = torch.Generator().manual_seed(7)
    bias = (torch.randn(n, generator=gen) * 30).to(dtype)
    held = (torch.randn(m, n, generator=gen) * 30).to(dtype)
    out = held.to(DEV)
    dionw.float8_product(a, b, bias=bias.to(DEV), out=out, accumulate=True)
    _close(out, a64, b64, bias.double() + held.double())
    room = torch.full((m + 2, n + 9), 5.0, dtype=dtype, device=DEV)
    _close(dionw.float8_product(a, b, out=room[1:-1, 3:n + 3]), a64, b64)
    assert bool((room[:, :3] == 5).all()) and bool((room[:, n + 3:] == 5).all()) and bool((room[[0, -1]] == 5).all())
    again = [dionw.float8_product(a, b, out_dtype=torch.float32) for _ in range(3)]
    assert torch.equal(again[0], again[1]) and torch.equal(again[0], again[2])


def test_product_of_nothing() -> None:
    a, _ = _operand(5, 256, False, 1)
    empty = Float8Matrix(a.values[:0], a.scales[:0])
    assert dionw.float8_product(empty, a).shape == (0, 5) and dionw.float8_product(a, empty).shape == (5, 0)
    none = Float8Matrix(a.values[:, :0], a.scales[:, :0])
    bias = torch.arange(5.0, device=DEV)
    for rows in (5, 200):
        left = Float8Matrix(torch.empty(rows, 0, dtype=torch.float8_e4m3fn, device=DEV), torch.empty(rows, 0, device=DEV))
        assert torch.equal(dionw.float8_product(left, none, bias=bias, out_dtype=torch.float32), bias.expand(rows, 5))


def test_product_nan_scales_reach_their_rows_alone() -> None:
    for m in (20, 150):
        a, _ = _operand(m, 256, False, 1)
        b, _ = _operand(140, 256, False, 2)
        a.scales[3, 1] = math.nan
        b.scales[130, 0] = math.nan
        bad = dionw.float8_product(a, b).isnan()
        expect = torch.zeros(m, 140, dtype=torch.bool, device=DEV)
        expect[3], expect[:, 130] = True, True
        assert torch.equal(bad, expect)


def test_product_is_the_same_each_time_on_streams_and_in_graphs() -> None:
    a, _ = _operand(700, 3000, False, 1)
    b, _ = _operand(900, 3000, True, 2)
    first = dionw.float8_product(a, b, out_dtype=torch.float32)
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    torch.cuda.synchronize()
    for stream in streams:
        with torch.cuda.stream(stream):
            results.append(dionw.float8_product(a, b, out_dtype=torch.float32))
    out = torch.empty_like(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dionw.float8_product(a, b, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(first, other) for other in (*results, out))
    from dionw_b200 import _native
    assert _native.device_status() == 0


# ---------------------------------------------------------------------------
# the linear layer
# ---------------------------------------------------------------------------
def _linear64(x: Tensor, w: Tensor, dy: Tensor, bias: Tensor | None):
    q = {"x": oracle.spread(*oracle.quantize(x, False)), "w": oracle.spread(*oracle.quantize(w, True)),
         "dy": oracle.spread(*oracle.quantize(dy, False)), "xt": oracle.spread(*oracle.quantize(x.T, False)),
         "dyt": oracle.spread(*oracle.quantize(dy.T, False))}
    return q


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 128, 256), (5, 100, 33), (130, 257, 140), (300, 512, 384)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear(tokens, inputs, outputs, dtype, with_bias) -> None:
    x, dy = _matrix(tokens, inputs, 1, dtype), _matrix(tokens, outputs, 2, dtype)
    w = _matrix(outputs, inputs, 3) * 0.1
    bias = torch.randn(outputs, generator=torch.Generator().manual_seed(4)) if with_bias else None
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, bias) if t is not None]
    y = dionw.float8_linear(*leaves)
    assert y.dtype is dtype
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    q = _linear64(x, w, dy, bias)
    _close(y.detach(), q["x"], q["w"], bias.double().expand(tokens, -1) if with_bias else 0.0)
    _close(grads[0], q["dy"], q["w"].T.contiguous())
    assert grads[1].dtype is torch.float32
    _close(grads[1], q["dyt"], q["xt"])
    if with_bias:
        want = dy.double().sum(0)
        assert bool(((grads[2].cpu().double() - want).abs() <= (tokens + 2) * 2.0**-24 * dy.double().abs().sum(0) + 1e-30).all())


@pytest.mark.parametrize("tokens,inputs,outputs", [(2501, 1900, 2405), (4097, 2304, 1281)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_many_tiles(tokens, inputs, outputs, dtype) -> None:
    """Enough tiles for the tensor cores to take the scales themselves."""
    x, dy = _matrix(tokens, inputs, 1, dtype).to(DEV).requires_grad_(), _matrix(tokens, outputs, 2, dtype).to(DEV)
    w = (_matrix(outputs, inputs, 3) * 0.1).to(DEV).requires_grad_()
    y = dionw.float8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    rows, columns = (q.dequantize().double() for q in dionw.quantize_rows(x, transposed=True))
    drows, dcolumns = (q.dequantize().double() for q in dionw.quantize_rows(dy, transposed=True))
    tiles, turned = (q.dequantize().double() for q in dionw.quantize_tiles(w, transposed=True))
    for got, a, b in ((y.detach(), rows, tiles), (dx, drows, turned), (dw, dcolumns, columns)):
        # one sum over the whole length on the tensor cores: a rounding of 2^-23 for each 32 products
        want, size = a @ b.T, a.abs() @ b.abs().T
        bound = (32 + a.shape[1] / 32) * 2.0**-23 * size + HALF_STEP[got.dtype] * 1.01 * want.abs() + 2.0**-25
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize("tokens,width", [(4096, 256), (4224, 256), (20000, 130), (9000, 2300)])
def test_long_sums_of_one_sign(tokens, width) -> None:
    """The weight's gradient over many tokens, all of it positive: what the tensor cores cut off in a piece of 32 blocks is
    128 times 2^-24 at most, and the pieces are added with a rounding each."""
    x, dy = _matrix(tokens, width, 1).abs().to(DEV), _matrix(tokens, width, 2).abs().to(DEV)
    w = torch.zeros(width, width, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad(dionw.float8_linear(x, w), w, dy)
    want = dionw.quantize_rows(dy, transposed=True)[1].dequantize().double() @ \
        dionw.quantize_rows(x, transposed=True)[1].dequantize().double().T
    pieces = -(-tokens // 4096)
    assert float(((dw.double() - want).abs() / want).max()) <= (128 + 4 + pieces) * 2.0**-24


def test_linear_of_many_tiles_keeps_infinities_in_their_rows() -> None:
    x = _matrix(2501, 1900, 1).to(DEV)
    w = (_matrix(2405, 1900, 3) * 0.1).to(DEV)
    clean = dionw.float8_linear(x, w)
    x[7, 3], x[2500, 1899], w[1000, 5] = math.inf, math.nan, math.nan
    y = dionw.float8_linear(x, w)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7], bad[2500], bad[:, 896:1024] = True, True, True
    assert torch.equal(y.isnan(), bad)
    assert torch.equal(y[~bad], clean[~bad])


def test_linear_gradients_are_those_of_differences() -> None:
    """The gradients against differences of the 64-bit layer in random directions.  Each quantized operand is off by at
    most 2^-4 of a value; errors of independent elements add up in squares, so that an inner product of 64 x 256
    terms is within a few percent of its size."""
    tokens, inputs, outputs = 64, 256, 128
    x, w, dy = _matrix(tokens, inputs, 5), _matrix(outputs, inputs, 6) * 0.1, _matrix(tokens, outputs, 7)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    grads = torch.autograd.grad(dionw.float8_linear(xs, ws), (xs, ws), dy.to(DEV))

    def loss(a: Tensor, b: Tensor) -> float:
        return float((a.double() @ b.double().T * dy.double()).sum())

    for leaf, grad in ((x, grads[0]), (w, grads[1])):
        direction = grad.cpu().double() / float(grad.double().norm())
        step = 1e-3 * float(leaf.norm())
        if leaf is x:
            difference = (loss(x + step * direction, w) - loss(x - step * direction, w)) / (2 * step)
        else:
            difference = (loss(x, w + step * direction) - loss(x, w - step * direction)) / (2 * step)
        assert difference == pytest.approx(float(grad.double().norm()), rel=0.05)


@pytest.mark.parametrize("rows,cols,shift", [(1, 1, 0), (0, 5, 0), (7, 33, 0), (1000, 130, 1), (33, 2000, 0), (4097, 64, 0)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_column_sums(rows, cols, shift, dtype) -> None:
    """A column's 64 partial sums are each of rows / 64 values: rows / 64 + 64 roundings of 2^-24."""
    from dionw_b200 import _native

    room = _matrix(rows, cols + shift + 3, 1, dtype).to(DEV)
    x = room[:, shift:cols + shift]
    out = torch.full((cols + 1,), 7.0, device=DEV)
    _native.on_device(0, _native.library().dionw_column_sums, x.data_ptr(), _native.dtype_code(dtype), rows, cols,
                      room.stride(0), out.data_ptr())
    want, size = x.double().sum(0), x.double().abs().sum(0)
    assert bool(((out[:cols].double() - want).abs() <= (rows / 64 + 66) * 2.0**-24 * size).all()) and float(out[cols]) == 7.0


def test_linear_of_any_leading_shape_and_partial_gradients() -> None:
    x = _matrix(24, 64, 8, torch.bfloat16).view(2, 3, 4, 64).to(DEV)
    layer = dionw.Float8Linear(64, 48, device=DEV)
    y = layer(x)
    assert y.shape == (2, 3, 4, 48) and y.dtype is torch.bfloat16
    y.float().sum().backward()
    assert layer.weight.grad.shape == (48, 64) and layer.weight.grad.dtype is torch.float32
    assert layer.bias.grad.shape == (48,)
    layer.weight.requires_grad_(False)
    leaf = x.clone().requires_grad_()
    layer(leaf).float().sum().backward()
    assert leaf.grad.shape == x.shape
    with torch.no_grad():
        assert not layer(x).requires_grad
    assert layer(x[:0]).shape == (0, 3, 4, 48)
    empty = x[:0].clone().requires_grad_()
    weight = torch.randn(48, 64, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(dionw.float8_linear(empty, weight).float().sum(), (empty, weight))
    assert dx.shape == empty.shape and float(dw.abs().max()) == 0.0
    with torch.autocast("cuda", torch.bfloat16):
        assert layer(x.float()).dtype is torch.bfloat16
    # no inputs: the bias alone
    bias = torch.randn(5, device=DEV)
    nothing = dionw.float8_linear(torch.zeros(2, 3, 0, device=DEV), torch.zeros(5, 0, device=DEV), bias)
    assert torch.equal(nothing, bias.expand(2, 3, 5))
    assert dionw.float8_linear(x[0, 0, 0], layer.weight).shape == (48,)


def test_linear_forward_and_backward_in_a_graph() -> None:
    x, w, dy = (t.to(DEV) for t in (_matrix(100, 256, 1, torch.bfloat16), _matrix(192, 256, 2), _matrix(100, 192, 3, torch.bfloat16)))
    x.requires_grad_(), w.requires_grad_()

    def once():
        y = dionw.float8_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    eager = [t.clone() for t in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, captured))
