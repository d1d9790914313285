"""The GELU of the 8-bit operators against x Phi(x) in 64 bits, over its whole range and its negative tail above all."""
import math

import pytest
import torch

from aitemplate_b200 import kernels
from test_int8_gpu import DTYPES, STEP32, _half_step

pytestmark = pytest.mark.gpu


def _gelu64(x):
    """(x Phi(x), how far 32 bits may be from it). The value is max(x, 0) - T with T = |x| Phi(-|x|) = 0.5 |x| exp(-z^2) t P(t). The polynomial is
    off by 8e-9 |x| at most, and by 3e-5 of T. In steps of 2^-24 of T: t three and a half (its sum, the constant, a reciprocal to 2^-23), times the
    2.35 that P answers with at most; P eight, its coefficients two; two products; exp four (2^-22) and three times its argument
    x^2 / 2. The last subtraction rounds once. What is under 2^-126 may be flushed."""
    t = 0.5 * x.abs() * torch.erfc(x.abs() * math.sqrt(0.5))  # (torch.special.ndtr gives 0 below -8.3 on the GPU)
    y = x.clamp(min=0) - t
    off = torch.minimum(8.1e-9 * x.abs(), 3.1e-5 * t) + t * STEP32 * (2.35 * 4 + 8 + 2 + 2 + 4 + 1.5 * x * x) + STEP32 * y.abs() + 2.0 ** -126
    return y, off


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_value(dtype):
    """A row of one value has that value's magnitude over 127 as its scale, in 32 bits."""
    x = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)]
    q, scale = kernels.quantize_rows(x[:, None], "gelu")
    want, off = _gelu64(x.double())
    assert bool((q[:, 0].double() == torch.where(scale > 0, 127 * torch.sign(x.double()), 0.0)).all())
    away = (scale.double() * 127 - want.abs()).abs()
    bound = off + STEP32 * want.abs() + 127 * 2.0 ** -150
    assert bool((away <= bound).all()), f"{float((away / bound).max()):.3f} of the bound"
    pairs = torch.stack([x, x], 1).contiguous()  # gated by itself
    want, off = want * x.double(), off * x.double().abs()
    small = (want.abs() < 3e38) & torch.isfinite(x.float() * x.float())
    _, scale = kernels.quantize_rows(pairs[small], "gelu", gated=True)
    away = (scale.double() * 127 - want[small].abs()).abs()
    assert bool((away <= off[small] + 2 * STEP32 * want[small].abs() + 2.0 ** -126 + 127 * 2.0 ** -150).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns,tile", [(1, 4096, 0), (9, 4096, 0), (4096, 8, 64), (4096, 64, 128), (4096, 24, 256), (4096, 512, 512), (4096, 9, 128)])
def test_as_an_epilogue(rows, columns, tile, dtype):
    """Results in 16 bits are right to their half step, small negative ones too. The sums are 1, the arguments the scales."""
    at = torch.linspace(-9, 5, max(rows, columns), device="cuda")
    x, w = torch.zeros(rows, 512, dtype=torch.int8, device="cuda"), torch.zeros(columns, 512, dtype=torch.int8, device="cuda")
    x[:, 3], w[:, 3] = 1, 1
    xs, ws = (at, torch.ones(columns, device="cuda")) if rows > columns else (torch.ones(rows, device="cuda"), at)
    y = kernels.gemm_rcr_i8(x, w, ws, xs, epilogue="gelu", dtype=dtype, tile_n=tile).double()
    want, off = _gelu64(xs.double()[:, None] * ws.double())
    bound = off + _half_step(dtype) * (want.abs() + off) + torch.finfo(dtype).smallest_normal * _half_step(dtype)
    assert bool(((y - want).abs() <= bound).all()), f"{float(((y - want).abs() / bound).max()):.3f} of the bound"
