"""Refusals of the 8-bit entry points; no GPU needed."""

from __future__ import annotations

from dionw_b200 import _native


def test_exponents_of_one_operand_are_refused() -> None:
    """They would go unused, and the product would be summed as one without."""
    lib = _native.library()
    at = 1 << 20   # an address that is never read

    def call(m: int, a_exponents: int | None, b_exponents: int | None) -> int:
        return lib.dionw_float8_product(at, 112, at, 1, m, 0, at, 112, at, 1, 6, 0, None, 0, at, 6, 0, 0, m, 6, 100, a_exponents,
                                        b_exponents, None, 0, None)

    for m in (0, 4, 200):
        for one in ((at, None), (None, at)):
            assert call(m, *one) == -1
            assert "one operand" in _native.last_error()
    assert call(0, at, at) == 0 and call(0, None, None) == 0
