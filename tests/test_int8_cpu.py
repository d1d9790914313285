"""What the 8-bit product, the quantisation of rows and the norms around a block refuse before they reach a GPU."""
import ctypes

import pytest
import torch

from aitemplate_b200 import _lib, kernels

F16, BF16, F32 = 1, 6, 2
P = ctypes.c_void_p(4096)  # a pointer that no refused call follows


def _refused(name, args, said):
    lib = _lib.load()
    assert getattr(lib, name)(*args) != 0
    assert said in _lib.last_error(), _lib.last_error()


def _gemm(a=P, a_scale=P, b=P, b_scale=P, bias=None, d0=None, d1=None, c=P, m=4, n=8, k=32, lda=32, ldb=32, ldc=8, ldd=8, epilogue=0,
          dtype=F16, tile_n=0):
    return [a, a_scale, b, b_scale, bias, d0, d1, c, m, n, k, lda, ldb, ldc, ldd, epilogue, dtype, tile_n, None]


@pytest.mark.parametrize("change,said", [
    (dict(k=131072, lda=131072, ldb=131072), "131071"), (dict(lda=31), "pitch"), (dict(ldb=16), "pitch"), (dict(ldc=7), "pitch"),
    (dict(epilogue=1 << 4, d0=P, ldd=4), "pitch"), (dict(epilogue=1 << 4), "needs d0"), (dict(epilogue=1 << 6, d0=P), "needs d1"),
    (dict(a_scale=None), "scales"), (dict(b_scale=None), "scales"), (dict(a=None), "null operand"), (dict(c=None), "null operand"),
    (dict(dtype=F32), "dtype"), (dict(m=-1), "negative"), (dict(k=0), "no columns"), (dict(c=ctypes.c_void_p(4097)), "aligned to its type"),
    (dict(bias=ctypes.c_void_p(4097)), "aligned to its type"), (dict(b_scale=ctypes.c_void_p(4098)), "aligned to its type"),
    (dict(a_scale=ctypes.c_void_p(4098)), "aligned to its type"),
])
def test_gemm_rcr_i8_refuses(change, said):
    _refused("b200ait_gemm_rcr_i8", _gemm(**change), said)


def test_gemm_rcr_i8_of_nothing():
    assert _lib.load().b200ait_gemm_rcr_i8(*_gemm(a=None, a_scale=None, c=None, m=0)) == 0
    assert _lib.load().b200ait_gemm_rcr_i8(*_gemm(b=None, b_scale=None, c=None, n=0)) == 0


def _x16(x=P, x_dtype=F16, b=P, b_scale=P, bias=None, d0=None, d1=None, c=P, m=8, n=8, k=32, ldx=32, ldb=32, ldc=8, ldd=8, epilogue=0,
         dtype=F16, tile_n=0, scratch=P, scratch_bytes=8 * 36):
    return [x, x_dtype, b, b_scale, bias, d0, d1, c, m, n, k, ldx, ldb, ldc, ldd, epilogue, dtype, tile_n, scratch, scratch_bytes, None]


@pytest.mark.parametrize("change,said", [
    (dict(x_dtype=F32), "x must be"), (dict(dtype=F32), "dtype"), (dict(scratch=None), "scratch"), (dict(scratch_bytes=8 * 36 - 1), "scratch"),
    (dict(scratch=ctypes.c_void_p(4104)), "scratch"), (dict(x=ctypes.c_void_p(4097)), "aligned to its type"), (dict(x=None), "null operand"),
    (dict(b_scale=None), "scales"), (dict(ldx=31), "pitch"), (dict(k=131072, ldx=131072, ldb=131072), "131071"), (dict(n=-1), "negative"),
])
def test_gemm_rcr_i8_x16_refuses(change, said):
    _refused("b200ait_gemm_rcr_i8_x16", _x16(**change), said)


def test_scratch_of_16_bit_rows():
    lib, out = _lib.load(), ctypes.c_int64(-1)
    for (m, n, k, ldb, b, tile), want in {(8, 8, 33, 48, 4096, 0): 8 * 48 + 32, (1, 8, 33, 48, 4096, 0): 0, (1, 8, 33, 40, 4096, 0): 52,
                                          (1, 8, 33, 48, 4104, 0): 52, (1, 8, 33, 48, 4096, 64): 52, (0, 8, 33, 48, 4096, 0): 0,
                                          (4, 4096, 4096, 4096, 4096, 0): 4 * 4100, (4, 1024, 1024, 1024, 4096, 0): 0}.items():
        assert lib.b200ait_gemm_rcr_i8_x16_scratch_bytes(b, m, n, k, ldb, tile, ctypes.byref(out)) == 0
        assert out.value == want, (m, n, k)


def _quantize(q=P, scale=P, x=P, rows=2, n=16, x_pitch=16, q_pitch=16, activation=0, gated=0, dtype=F16):
    return [q, scale, x, rows, n, x_pitch, q_pitch, activation, gated, dtype, None]


@pytest.mark.parametrize("change,said", [
    (dict(dtype=F32), "dtype"), (dict(rows=-1), "negative"), (dict(activation=8), "activation"), (dict(activation=-1), "activation"),
    (dict(x=None), "null"), (dict(scale=None), "null"), (dict(x_pitch=15), "pitch"), (dict(q_pitch=15), "pitch"),
    (dict(gated=1), "pitch"), (dict(rows=1 << 31), "int32"), (dict(x=ctypes.c_void_p(4097)), "aligned to its type"),
    (dict(scale=ctypes.c_void_p(4098)), "aligned to its type"),
])
def test_quantize_rows_refuses(change, said):
    _refused("b200ait_quantize_rows", _quantize(**change), said)


def _norm(sum=P, y=P, y_scale=None, x=P, residual=None, gate=None, post_gamma=None, post_beta=None, gamma=None, beta=None, rows=6, n=16,
          gates=1, gammas=1, betas=1, y_pitch=16, post_norm=0, norm=1, residual_scale=1.0, eps=1e-5, dtype=BF16):
    return [sum, y, y_scale, x, residual, gate, post_gamma, post_beta, gamma, beta, rows, n, gates, gammas, betas, y_pitch, post_norm, norm,
            residual_scale, eps, dtype, None]


@pytest.mark.parametrize("change,said", [
    (dict(dtype=F32), "dtype"), (dict(norm=0), "layer (1) or rms (2)"), (dict(norm=3), "layer (1) or rms (2)"), (dict(post_norm=3), "none (0)"),
    (dict(post_gamma=P), "need a norm"), (dict(x=None), "null"), (dict(y=None), "null"), (dict(gate=P, gates=4), "each gate"),
    (dict(gamma=P, gammas=0), "each gamma"), (dict(beta=P, betas=5), "each beta"), (dict(y_scale=P, y_pitch=8), "pitch"), (dict(n=-1), "negative"),
    (dict(gamma=ctypes.c_void_p(4097)), "aligned to its type"), (dict(y=ctypes.c_void_p(4097)), "aligned to its type"),
    (dict(y_scale=ctypes.c_void_p(4098)), "aligned to its type"),
])
def test_residual_norm_refuses(change, said):
    _refused("b200ait_residual_norm", _norm(**change), said)


def test_cpu_tensors_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    x, w, s = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: kernels.gemm_rcr_i8(x, w, s, s[:2]), lambda: kernels.quantize_rows(x.half()), lambda: kernels.residual_norm(x.half())):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()


@pytest.mark.parametrize("shape,strides,pitch", [
    ((5, 7), (16, 1), 16), ((1, 7), (99, 1), 7), ((2, 3, 8), (48, 16, 1), 16), ((2, 1, 8), (48, 5, 1), 48), ((8,), (1,), 8), ((4, 1), (3, 9), 3),
])
def test_row_pitch(shape, strides, pitch):
    assert kernels._row_pitch("f", "x", torch.zeros(1000).as_strided(shape, strides)) == pitch


@pytest.mark.parametrize("shape,strides", [((5, 7), (7, 2)), ((5, 7), (6, 1)), ((2, 3, 8), (40, 16, 1)), ((2, 3, 8), (0, 8, 1))])
def test_rows_that_have_no_pitch(shape, strides):
    with pytest.raises(ValueError, match="f: "):
        kernels._row_pitch("f", "x", torch.zeros(1000).as_strided(shape, strides))
