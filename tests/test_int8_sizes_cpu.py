"""Sizes at the end of 32 bits: past the last row and column the kernels of 8-bit products count on, and that must not wrap."""
import pytest
import torch  # noqa: F401 (its CUDA libraries)

from test_int8_cpu import _gemm, _refused, _x16

END = 1 << 31


@pytest.mark.parametrize("change", [dict(n=END - 1, ldc=END, ldd=END), dict(n=END - 1023, ldc=END, ldd=END), dict(m=END - 1), dict(m=1, n=END - 1, ldc=END, ldd=END)])
def test_products_that_would_count_past_32_bits(change):
    _refused("b200ait_gemm_rcr_i8", _gemm(**change), "int32")
    _refused("b200ait_gemm_rcr_i8_x16", _x16(**{**change, "scratch_bytes": 1 << 40}), "int32")
