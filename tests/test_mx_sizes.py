"""Sizes of MXFP4 operands that the C-ABI takes or refuses before any launch, at the ends of their ranges."""

import pytest

from comp_b200 import _lib, mx

MOST_ROWS, MOST_K = 2**31 - 1 - 1024, 2**30 - 32


@pytest.mark.parametrize("experts,rows,k", [(1024, MOST_ROWS, MOST_K), (1024, 1 << 30, 1 << 29), (512, MOST_ROWS, 1 << 27),
                                            (1024, MOST_ROWS, 1 << 25), (8, MOST_ROWS, MOST_K), (7, MOST_ROWS, MOST_K),
                                            (1, MOST_ROWS, MOST_K), (1024, MOST_ROWS, 1 << 22), (1024, 1, MOST_K)])
def test_bytes_past_64_bits(experts, rows, k):
    """An operand's bytes are the ones that it takes, or it is refused by all that would handle it."""
    lib, true = _lib.load(), mx.image_bytes(rows, k, experts)
    if true < 1 << 63:
        assert lib.b2q_mx_bytes(experts, rows, k) == true
        return
    assert lib.b2q_mx_bytes(experts, rows, k) == 0 and "b2q_mx_bytes" in _lib.last_error()
    for call in (lambda: lib.b2q_mx_quantize(0, 4096, k, experts, rows, k, 4096, None),
                 lambda: lib.b2q_mx_dequantize(4096, experts, rows, k, 0, 4096, k, None),
                 lambda: lib.b2q_mx_pack(4096, 4096, experts, rows, k, 4096, None)):
        assert call() == -4 and "64-bit" in _lib.last_error()
