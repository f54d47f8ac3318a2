"""What the 8-bit entry points refuse, and their oracle; no GPU needed."""

from __future__ import annotations

import math

import pytest
import torch

import dionw_b200 as dionw
from dionw_b200 import Float8Matrix, _native
from dionw_b200.adamw8 import dequantize_moments
from oracle import eight_bit as oracle

E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# the formats and the oracle's rounding
# ---------------------------------------------------------------------------
def test_format_values_are_torchs() -> None:
    for values, dtype in ((oracle.E4M3, torch.float8_e4m3fn), (oracle.E5M2, torch.float8_e5m2)):
        codes = torch.arange(len(values), dtype=torch.uint8).view(dtype)
        assert torch.equal(codes.double(), values)


def test_oracle_quantizes_as_torch_rounds() -> None:
    x = torch.randn(130, 300, generator=torch.Generator().manual_seed(0))
    values, scales = oracle.quantize(x, False)
    expect = (x.double() / scales.repeat_interleave(128, 1)[:, :300]).float().to(E4M3).double()
    assert torch.equal(values, expect)
    assert float(values.abs().max()) <= 448.0 and float(values.abs().amax()) > 224.0


def test_stochastic_code_is_right_on_average_and_exact_on_codes() -> None:
    codes = torch.arange(127)
    everywhere = torch.tensor([0, 1, 65535])
    for part in everywhere:
        assert torch.equal(oracle.stochastic_code(oracle.E4M3, oracle.E4M3, part.expand(127)), codes)
    x = torch.full((65536,), 1.03, dtype=torch.float64)
    mean = oracle.E4M3[oracle.stochastic_code(x, oracle.E4M3, torch.arange(65536))].mean()
    assert float(mean) == pytest.approx(1.03, abs=0.125 / 65536)


def test_noise_words_differ_by_element_step_and_seed() -> None:
    index = torch.arange(4096)
    words = [oracle.noise(index, 1, 0), oracle.noise(index, 2, 0), oracle.noise(index, 1, 1),
             oracle.noise(index + 2**32, 1, 0)]
    for i, a in enumerate(words):
        assert 0 <= int(a.min()) and int(a.max()) < 2**32
        assert abs(float((a % 65536).double().mean()) / 32767.5 - 1) < 0.05
        assert abs(float((a // 65536).double().mean()) / 32767.5 - 1) < 0.05
        for b in words[:i]:
            assert float((a == b).double().mean()) < 0.01


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def _adamw8_args(n: int = 256) -> list[list[torch.Tensor]]:
    p = torch.zeros(n)
    state = dionw.adamw8_state(p)
    return [[p], [torch.zeros(n)], [state["exp_avg"]], [state["exp_avg_sq"]], [state["exp_avg_scale"]],
            [state["exp_avg_sq_scale"]], [state["adamw_step"]]]


def test_adamw8_state_is_zero_and_dequantizes() -> None:
    state = dionw.adamw8_state(torch.zeros(3, 50))
    assert {key: (tuple(t.shape), t.dtype) for key, t in state.items()} == {
        "exp_avg": ((3, 50), torch.float8_e4m3fn), "exp_avg_sq": ((3, 50), torch.float8_e5m2),
        "exp_avg_scale": ((2,), torch.float32), "exp_avg_sq_scale": ((2,), torch.float32),
        "adamw_step": ((), torch.float32)}
    state["exp_avg"].view(-1)[130] = 2.0
    state["exp_avg_scale"][1] = 3.0
    mean, square = dequantize_moments(state)
    assert float(mean.view(-1)[130]) == 6.0 and float(mean.sum()) == 6.0 and float(square.sum()) == 0.0


def test_adamw8_step_refuses() -> None:
    step = dionw.adamw8_step
    args = _adamw8_args()
    with pytest.raises(ValueError, match="CUDA"):
        step(*args, lr=1e-3)
    step(*[[] for _ in args], lr=1e-3)   # nothing to do
    with pytest.raises(ValueError, match="1 parameters"):
        step(*args[:6], [], lr=1e-3)
    for more, match in (({"betas": (1.0, 0.9)}, "betas"), ({"betas": (0.9, -0.1)}, "betas"), ({"eps": 0.0}, "eps"),
                        ({"lr": -1.0}, "lr"), ({"lr": math.nan}, "lr"), ({"weight_decay": math.inf}, "weight_decay"),
                        ({"seed": -1}, "seed"), ({"seed": 2**32}, "seed")):
        with pytest.raises(ValueError, match=match):
            step(*args, **{"lr": 1e-3, **more})


def test_adamw8_entry_refuses() -> None:
    lib = _native.library()
    call = [None, None, 0, None, None, None, None, None, None, 0, 1e-3, 0.9, 0.95, 0.0, 1e-8, 0, None, None]
    assert lib.dionw_adamw8_multi(*call) == 0
    for at, value, match in ((9, -1, "tensor count"), (2, 3, "dtype"), (11, 1.0, "betas"), (12, -0.5, "betas")):
        bad = list(call)
        bad[at] = value
        assert lib.dionw_adamw8_multi(*bad) == -1
        assert match in _native.last_error()


def test_quantize_refuses() -> None:
    for quantize in (dionw.quantize_rows, dionw.quantize_tiles):
        with pytest.raises(ValueError, match="matrix"):
            quantize(torch.zeros(3))
        with pytest.raises(ValueError, match="CUDA"):
            quantize(torch.zeros(3, 4))


def test_quantize_entry_refuses() -> None:
    lib = _native.library()
    # an address that is never read: every call below is refused, or has nothing to do
    at, off = 1 << 20, (1 << 20) + 8

    def call(x=at, dtype=0, rows=4, cols=100, ldx=100, q=at, ldq=112, scales=at, lds=4, qt=None, ldqt=0, scales_t=None,
             ldst=0):
        return lib.dionw_float8_quantize(x, dtype, rows, cols, ldx, 0, q, ldq, scales, lds, qt, ldqt, scales_t, ldst, None, None,
                                         None)

    assert call(rows=0) == 0 and call(cols=0) == 0
    for bad, match in ((dict(dtype=3), "dtype"), (dict(rows=-1), "shape"), (dict(ldx=99), "leading dimension"),
                       (dict(x=None), "leading dimension"), (dict(q=None), "nothing to write"), (dict(q=off), "16-byte"),
                       (dict(ldq=100), "16-byte"), (dict(ldq=96), "16-byte"), (dict(scales=None), "scale"),
                       (dict(lds=3), "scale"), (dict(qt=off, ldqt=16, scales_t=at, ldst=100), "transposed"),
                       (dict(qt=at, ldqt=0, scales_t=at, ldst=100), "transposed"),
                       (dict(qt=at, ldqt=16, scales_t=at, ldst=99), "transposed"), (dict(rows=1 << 30), "rows")):
        assert call(**bad) == -1, bad
        assert match in _native.last_error(), (bad, _native.last_error())


def _float8(rows: int, cols: int, tiles: bool = False) -> Float8Matrix:
    room = torch.zeros(rows, (cols + 15) // 16 * 16).to(E4M3)
    return Float8Matrix(room[:, :cols], torch.ones(-(-rows // 128) if tiles else rows, -(-cols // 128)))


def test_float8_matrix_refuses() -> None:
    good = _float8(4, 200)
    assert good.shape == (4, 200) and not good.tiles and _float8(4, 200, True).tiles
    assert torch.equal(good.dequantize(), torch.zeros(4, 200))
    with pytest.raises(TypeError):
        Float8Matrix(good.values.float(), good.scales)
    with pytest.raises(TypeError):
        Float8Matrix(good.values, good.scales.half())
    with pytest.raises(ValueError, match="two matrices"):
        Float8Matrix(good.values[0], good.scales)
    with pytest.raises(ValueError, match="fit neither"):
        Float8Matrix(good.values, good.scales[:3])
    with pytest.raises(ValueError, match="fit neither"):
        Float8Matrix(good.values, good.scales[:, :1])
    with pytest.raises(ValueError, match="16-byte"):
        Float8Matrix(good.values[:, 1:130], good.scales)
    with pytest.raises(ValueError, match="16-byte"):
        Float8Matrix(torch.zeros(4, 200).to(E4M3), good.scales)     # 200 bytes apart
    with pytest.raises(ValueError, match="16-byte"):
        Float8Matrix(torch.zeros(200, 4).to(E4M3).T, good.scales)


def test_float8_product_refuses() -> None:
    a, b = _float8(4, 200), _float8(6, 200)
    with pytest.raises(ValueError, match="CUDA"):
        dionw.float8_product(a, b)
    with pytest.raises(ValueError, match="columns"):
        dionw.float8_product(a, _float8(6, 100))


def test_float8_product_entry_refuses() -> None:
    lib = _native.library()
    at, off = 1 << 20, (1 << 20) + 4

    def call(a=at, lda=112, sa=at, b=at, ldb=112, sb=at, bias=None, bias_dtype=0, out=at, ldo=6, out_dtype=0, m=4, n=6, k=100):
        return lib.dionw_float8_product(a, lda, sa, 1, 4, 0, b, ldb, sb, 1, 6, 0, bias, bias_dtype, out, ldo, out_dtype, 0,
                                        m, n, k, None, None, None, 0, None)

    assert call(m=0) == 0 and call(n=0) == 0
    for bad, match in ((dict(m=-1), "shape"), (dict(k=1 << 33), "shape"), (dict(out_dtype=3), "output"),
                       (dict(bias=at, bias_dtype=-1), "bias"), (dict(out=None), "leading"), (dict(ldo=5), "leading"),
                       (dict(a=None), "null"), (dict(sb=None), "null"), (dict(a=off), "16-byte"), (dict(b=off), "16-byte"),
                       (dict(lda=100), "16-byte"), (dict(ldb=104), "16-byte"), (dict(ldb=96), "16-byte")):
        assert call(**bad) == -1, bad
        assert match in _native.last_error(), (bad, _native.last_error())


def test_float8_product_scratch() -> None:
    lib = _native.library()
    assert lib.dionw_float8_product_workspace_bytes(64, 4096, 4096) == 0
    assert lib.dionw_float8_product_workspace_bytes(0, 1 << 20, 8) == 0
    assert lib.dionw_float8_product_workspace_bytes(1 << 14, 1 << 14, 0) == 0
    # 296 words, and 512 bytes for each 128 rows and block of both operands
    assert lib.dionw_float8_product_workspace_bytes(8192, 14336, 4096) == 1536 + 512 * 32 * (64 + 112)
    status = lib.dionw_float8_product(1 << 20, 4096, 1 << 20, 1, 8192, 0, 1 << 20, 4096, 1 << 20, 1, 14336, 0, None, 0, 1 << 20,
                                      14336, 0, 0, 8192, 14336, 4096, None, None, 1 << 20, 100, None)
    assert status == -3 and "workspace" in _native.last_error()


def test_float8_linear_refuses() -> None:
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    with pytest.raises(ValueError, match="CUDA"):
        dionw.float8_linear(x, w)
    with pytest.raises(ValueError, match="does not fit"):
        dionw.float8_linear(x, w.T)
    with pytest.raises(ValueError, match="does not fit"):
        dionw.float8_linear(x, w[0])
    with pytest.raises(TypeError, match="x is"):
        dionw.float8_linear(x.long(), w)
    layer = dionw.Float8Linear(8, 5)
    groups, report = dionw.param_groups(torch.nn.Sequential(torch.nn.Linear(64, 64), dionw.Float8Linear(64, 64)))
    assert [g["dion_route"] for g in groups] == ["adamw", "matrix"] and len(groups[1]["params"]) == 2
    assert isinstance(layer, torch.nn.Linear)


# ---------------------------------------------------------------------------
# Dion's option
# ---------------------------------------------------------------------------
def test_dion_state_bits_are_checked() -> None:
    from dionw_b200._keys import ADAMW_STATE_BITS_KEY
    from dionw_b200.optimizer import _require_group, _require_same_structure

    assert ADAMW_STATE_BITS_KEY == "adamw_state_bits"
    with pytest.raises(ValueError, match="adamw_state_bits must be 8 or 32"):
        dionw.Dion([], lr=1e-3, adamw_state_bits=16)
    common = {"params": [], "newton_schulz": "gram", "row_normalization": "normuon", "momentum_form": "heavy_ball",
              "lr": 1e-3, "weight_decay": 0.0, "fraction": 1.0, "num_heads": None}
    for bits in (8, 32):
        _require_group({**common, "dion_route": "adamw", "adamw_state_bits": bits})
    with pytest.raises(ValueError, match="must be 8 or 32"):
        _require_group({**common, "dion_route": "adamw", "adamw_state_bits": 4})
    with pytest.raises(ValueError, match="matrix group"):
        _require_group({**common, "dion_route": "matrix", "adamw_state_bits": 8})
    plain = {**common, "dion_route": "adamw"}
    _require_same_structure([plain], [{**plain, "adamw_state_bits": 32}])
    for old, new in ((8, 32), (32, 8)):
        with pytest.raises(ValueError, match="checkpoint=%d, optimizer=%d" % (old, new)):
            _require_same_structure([{**plain, "adamw_state_bits": old}], [{**plain, "adamw_state_bits": new}])


def test_a_step_of_tensors_elsewhere_or_of_other_moments_is_refused() -> None:
    from dionw_b200._adamw import adamw_step, init_adamw_state

    param = torch.zeros(300, requires_grad=True)
    param.grad = torch.ones(300)
    group = {"params": [param], "lr": 1e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0}
    state: dict = {param: dionw.adamw8_state(param)}
    with pytest.raises(ValueError, match="one CUDA device"):
        adamw_step({**group, "adamw_state_bits": 8}, state)
    with pytest.raises(ValueError, match="cannot change"):
        adamw_step(group, state)
    state[param] = {}
    init_adamw_state(param, state[param])
    with pytest.raises(ValueError, match="cannot change"):
        adamw_step({**group, "adamw_state_bits": 8}, state)


def test_tensor_table_is_what_torch_says() -> None:
    x = torch.randn(6, 50)
    tensors = [x, torch.nn.Parameter(x), x.to(E4M3), x.to(torch.float8_e5m2), x.half(), x.bfloat16(), x.T, x[1:], x.view(-1)[7:],
               x[:, :1], x[:, ::2], torch.zeros(()), torch.zeros(0, 5), torch.zeros(1, 4, 1), x.expand(3, 6, 50), x[:, None]]
    addresses, numels, kinds = _native.tensor_table(tensors)
    assert list(addresses) == [t.data_ptr() for t in tensors] and list(numels) == [t.numel() for t in tensors]
    for t, kind in zip(tensors, kinds):
        assert bool(kind >> 48) == t.is_contiguous(), t.shape
        # on CPU: device type 1
        assert kind % 2**32 == _native.tensor_kind(t.dtype, 0) % 2**32 and kind >> 32 & 0xFFFF == 1
    assert len(set(_native.tensor_kind(t, d) for t in _native._DL_TYPES for d in range(8))) == 8 * len(_native._DL_TYPES)
    assert all(len(values) == 0 for values in _native.tensor_table([]))
    for bad in (3, None, x.to_sparse(), torch.zeros(3, device="meta")):
        with pytest.raises(TypeError, match="memory of their own"):
            _native.tensor_table([x, bad])


def test_lists_and_room_that_are_missing_are_refused() -> None:
    lib = _native.library()
    at = 1 << 20
    assert lib.dionw_adamw8_multi(at, at, 0, at, at, at, at, None, at, 1, 1e-3, 0.9, 0.95, 0.0, 1e-8, 0, None, None) == -1
    assert "null list" in _native.last_error()
    assert lib.dionw_float8_linear_forward(at, 0, 8, at, 0, 8, None, 0, at, 4, 8, 8, None, None, None, None) == -1
    assert "room" in _native.last_error()
    assert lib.dionw_float8_linear_forward(at, 0, 8, at, 0, 8, None, 0, at, 4, 8, 8, at, at + 8, None, None) == -1
    assert "room" in _native.last_error()
    assert lib.dionw_float8_linear_backward(at, 0, 8, at, 0, None, 0, None, 4, 8, 8, None, None, at, None) == -1
    assert "room" in _native.last_error()


def test_linear_entries_refuse() -> None:
    lib = _native.library()
    at = 1 << 20
    assert lib.dionw_float8_packed_bytes(-1, 4, 0) == 0 and lib.dionw_float8_packed_bytes(0, 0, 0) == 256
    # codes 130 x 304, scales 3 x 130, exponents 3 x 2 x 128, each from a multiple of 256 bytes on
    assert lib.dionw_float8_packed_bytes(130, 300, 0) == 39680 + 1792 + 6 * 512
    assert lib.dionw_float8_packed_bytes(130, 300, 1) == 39680 + 256 + 6 * 512
    assert lib.dionw_float8_linear_forward(at, 0, 8, at, 0, 8, None, 0, at, -1, 8, 8, at, None, None, None) == -1
    assert "bad shape" in _native.last_error()
    assert lib.dionw_float8_linear_backward(at, 0, 8, at, 0, None, 0, None, 4, 8, 8, at, None, None, None) == -1
    assert "keeps" in _native.last_error()
    assert lib.dionw_float8_linear_backward(at, 0, 8, None, 0, at, 0, None, 4, 8, 8, at, None, at, None) == -1
    assert lib.dionw_column_sums(None, 0, 0, 0, 0, None, None) == 0
    for call in ((at, 3, 4, 8, 8, at, None), (at, 0, -1, 8, 8, at, None), (None, 0, 4, 8, 8, at, None),
                 (at, 0, 4, 8, 7, at, None), (at, 0, 4, 8, 8, None, None)):
        assert lib.dionw_column_sums(*call) == -1
        assert "column_sums" in _native.last_error()
