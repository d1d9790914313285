"""Gated rows whose products lie under 2^-126 are quantised by every kernel, those of rows past the registers of a block among them."""
import pytest
import torch

from aitemplate_b200 import kernels
from test_int8_gpu import STEP32, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 1001, 20001, 32768, 33000])
def test_small_gated_products(n):
    x = (torch.randn(3, 2 * n, generator=_gen(n), device="cuda") * 2.0 ** -66).to(torch.bfloat16)
    q, scale = kernels.quantize_rows(x, gated=True)
    v = (x[:, :n].double() * x[:, n:].double())
    v32 = x[:, :n].float() * x[:, n:].float()  # (torch keeps small values too)
    assert bool((v.abs().amax(1) < 2.0 ** -126).all())
    most = v32.double().abs().amax(1)
    assert bool(((scale.double() - most / 127).abs() <= STEP32 * most / 127 + 2.0 ** -150).all())
    # the products are whole steps of 2^-149, and 127 of the largest one's steps are those of q
    away = (q.double() - 127 * v / v.abs().amax(1, keepdim=True)).abs()
    assert bool((away <= 0.5 + 127 * 2 * 2.0 ** -150 / most[:, None] + 1e-4).all())
    assert bool((q.abs().amax(1) == 127).all())
