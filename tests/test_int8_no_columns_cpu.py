"""Rows without columns have no scale: a call that would have to write one is refused, one that has nothing to write is not."""
from aitemplate_b200 import _lib
from test_int8_cpu import P, _norm, _quantize, _refused


def test_rows_without_columns():
    _refused("b200ait_quantize_rows", _quantize(n=0), "no columns")
    _refused("b200ait_quantize_rows", _quantize(n=0, gated=1), "no columns")
    _refused("b200ait_residual_norm", _norm(n=0, y_scale=P), "no columns")
    assert _lib.load().b200ait_quantize_rows(*_quantize(rows=0, n=0)) == 0
    assert _lib.load().b200ait_residual_norm(*_norm(n=0)) == 0
    assert _lib.load().b200ait_residual_norm(*_norm(rows=0, n=0, y_scale=P)) == 0
