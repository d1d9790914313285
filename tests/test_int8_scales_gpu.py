"""gemm_rcr_i8 with scales that are no normal numbers (rows of bf16 values under 2^-119 have such): every kernel takes them as they are."""
import pytest
import torch

from aitemplate_b200 import kernels
from test_int8_gpu import _close, _gen, _product64

pytestmark = pytest.mark.gpu

# CUDA cores, weight streaming, tiles of every width, results that TMA cannot describe, rows off 16 bytes
PROBLEMS = [(1, 64, 512, 0), (2, 64, 512, 0), (9, 256, 512, 0), (9, 259, 512, 0), (70, 64, 512, 64), (70, 264, 512, 128), (300, 264, 512, 256),
            (300, 512, 512, 512), (70, 131, 512, 128), (20, 40, 33, 0)]


@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
@pytest.mark.parametrize("row,column", [(1e-39, 1.0), (1.0, 1e-39), (1e-39, 1e6), (3e-43, 1.0), (1e-20, 1e-19)])
def test_small_scales(m, n, k, tile, row, column):
    g = _gen(m + n)
    x, w = (torch.randint(1, 100, (r, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8) for r in (m, n))
    xs, ws = torch.full((m,), row, device="cuda"), torch.full((n,), column, device="cuda")
    bias = torch.full((n,), 1e-36, device="cuda").to(torch.bfloat16)
    for b, epilogue in ((None, ""), (bias, ""), (None, "add_relu")):
        d0 = torch.full((m, n), -1e-37, device="cuda").to(torch.bfloat16) if epilogue else None
        y = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, d0=d0, epilogue=epilogue, dtype=torch.bfloat16, tile_n=tile)
        want, off = _product64(x, w, xs, ws, b, d0, None, epilogue)
        # (behind the scales the arithmetic flushes what is under 2^-126, here as for 16-bit operands: with a residual, such sums)
        _close(y, want, off + (2.0 ** -126 if epilogue else 0.0), torch.bfloat16)


def test_small_rows():
    """The same from 16-bit values: quantised, and quantised on the way."""
    for m, n, k in ((1, 64, 512), (3, 64, 512), (9, 256, 512), (70, 131, 512), (300, 1000, 512)):
        x = (torch.randn(m, k, generator=_gen(m), device="cuda") * 2.0 ** -126).to(torch.bfloat16)
        w = torch.randint(1, 100, (n, k), generator=_gen(n), device="cuda", dtype=torch.int32).to(torch.int8)
        ws = torch.ones(n, device="cuda")
        q, scale = kernels.quantize_rows(x)
        assert bool((scale < 2.0 ** -126).all()) and bool((scale > 0).all())
        y = kernels.gemm_rcr_i8(q, w, ws, scale, dtype=torch.bfloat16)
        want, off = _product64(q, w, scale, ws, None, None, None, "")
        _close(y, want, off + 2.0 ** -149, torch.bfloat16)  # (a result may be small itself: its step is 2^-149 in 32 bits)
        assert torch.equal(kernels.gemm_rcr_i8(x, w, ws, dtype=torch.bfloat16), y)
