"""The 8-bit operators where a CTA or a thread does more than one piece of work: several tiles to a CTA, several units of a gated or activated row to a
thread, offsets past 32 bits, calls side by side."""
import pytest
import torch

from aitemplate_b200 import kernels
from test_int8_gpu import (DTYPES, MANY, STEP32, _act64, _act_off, _at, _close, _gen, _near_quantized, _norm_operands, _problem, _product64,
                           _quantized64, _residual_norm64, _weights)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epilogue,bias", [("", False), ("", True), ("gelu", True), ("add", False), ("add", True), ("mul_add", True), ("sigmoid_mul", False)])
@pytest.mark.parametrize("n", [5128, 5129])
def test_several_tiles_to_a_cta(n, epilogue, bias):
    """5 tiles to a pair of CTAs and up to 18 to a CTA, with column scales that differ from one block of 64 columns to the next: a tile that took
    another one's scales, bias or sums would show. Sums are exact and scaled in one order, so every width gives the same."""
    m, k, dtype = 4100, 128, DTYPES[(n + bias) % 2]
    x, w, ws, xs, b, d0, d1 = _problem(m, n, k, dtype, epilogue, bias, n)
    ws = ws * 4.0 ** ((torch.arange(n, device="cuda") // 64) % 5 - 2)
    want, off = _product64(x, w, xs, ws, b, d0, d1, epilogue)
    first = None
    for tile in (64, 128, 256, 512, 0):
        y = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, d0=d0, d1=d1, epilogue=epilogue, dtype=dtype, tile_n=tile)
        if first is None:
            first = y
            _close(y, want, off, dtype)
        assert torch.equal(y, first), tile
    assert kernels.device_status() == 0


@pytest.mark.parametrize("n", MANY)
def test_many_gated_rows(n):
    """Every number of units a thread of gated rows and of activated ones; where n is no multiple of 8 the second half lies elsewhere in 16 bytes."""
    activations = ("identity", "relu", "gelu", "fast_gelu", "sigmoid", "tanh", "swish", "hardswish")
    for i, gated in enumerate((True, True, False)):
        activation, dtype = activations[(n // 8 + 3 * i) % 8], DTYPES[(n // 8 + i) % 2]
        x = torch.randn(601, n * (2 if gated else 1), generator=_gen(n + i), device="cuda").to(dtype)
        q, scale = kernels.quantize_rows(x, activation, gated=gated)
        g = x[:, :n].double()
        v, off = _act64(activation, g), _act_off(activation, g, STEP32 * g.abs())
        if gated:
            u = x[:, n:].double()
            v, off = v * u, (off + STEP32 * v.abs()) * u.abs()
        _near_quantized(q, scale, v, off)


@pytest.mark.parametrize("n", [8200, 12001, 16384, 20001, 24571, 32768])
def test_wide_gated_rows(n):
    for rows, activation, dtype in ((1, "gelu", torch.float16), (7, "swish", torch.bfloat16)):
        x = torch.randn(rows, 2 * n, generator=_gen(n), device="cuda").to(dtype)
        q, scale = kernels.quantize_rows(x, activation, gated=True)
        g, u = x[:, :n].double(), x[:, n:].double()
        v, off = _act64(activation, g), _act_off(activation, g, STEP32 * g.abs())
        _near_quantized(q, scale, v * u, (off + STEP32 * v.abs()) * u.abs())


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 6, 7])
def test_narrow_rows(n):
    """Rows shorter than what a 16-byte piece of memory holds, at every place of 16 bytes."""
    for rows in (1, 2, 3, 5, 9, 30):
        for place in range(8):
            x = _at(torch.randn(rows, n, generator=_gen(rows), device="cuda").half(), place)
            q, scale = kernels.quantize_rows(x)
            want, ws = _quantized64(x.double())
            assert torch.equal(q.double(), want) and bool(((scale.double() - ws).abs() <= STEP32 * ws).all())
            both = _at(torch.cat([x, x.flip(1)], 1), place)
            q, scale = kernels.quantize_rows(both, "relu", gated=True)
            v = x.double().clamp(min=0) * x.flip(1).double()
            _near_quantized(q, scale, v, STEP32 * v.abs())
        x, o = _norm_operands(rows, n, torch.float16, n, 1, None, "rms")
        (total, off_t), (want, off_y) = _residual_norm64(x, o)
        for place in range(8):
            s, y = kernels.residual_norm(_at(x, place), **{**o, "residual": _at(o["residual"], place)})
            _close(s, total, off_t, torch.float16)
            _close(y, want, off_y, torch.float16)


def test_offsets_past_32_bits():
    """More than 2^31 elements to an operand: the last rows are what they are alone."""
    rows, n = 70001, 32768
    g = _gen(1)
    x = torch.randn(rows, n, generator=g, device="cuda", dtype=torch.float16)
    for f in (lambda t: kernels.quantize_rows(t), lambda t: kernels.quantize_rows(t, "swish", gated=True), lambda t: kernels.residual_norm(t, t, norm="rms"),
              lambda t: kernels.residual_norm(t, t, post_norm="rms", quantize=True)):
        some = f(x)
        alone = f(x[-3:])
        for a, b in zip(some, alone):
            assert torch.equal(a[-3:], b)
        del some
    odd = x.view(-1)[:70001 * 32765].view(70001, 32765)
    a, b = kernels.quantize_rows(odd), kernels.quantize_rows(_at(odd[-2:], 70001 * 32765 % 8 - 2 * 32765 % 8))
    assert torch.equal(a[0][-2:], b[0]) and torch.equal(a[1][-2:], b[1])
    del x, odd, a, b
    for n in (60000, 60001):
        m, k = 40000, 64
        x, w, ws, xs, b, d0, _ = _problem(m, n, k, torch.float16, "add", True, n)
        y = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, d0=d0, epilogue="add")
        assert torch.equal(y[-200:], kernels.gemm_rcr_i8(x[-200:], w, ws, xs[-200:], bias=b, d0=d0[-200:], epilogue="add"))
        want, off = _product64(x[-20:], w, xs[-20:], ws, b, d0[-20:], None, "add")
        _close(y[-20:], want, off, torch.float16)
        del x, w, d0, y
    torch.cuda.empty_cache()


def test_16_bit_rows_captured_and_side_by_side():
    """Rows quantised into scratch by calls on two streams at once, and by two graphs that are replayed in turn and at once: each has its own."""
    m, n, k = 300, 520, 1001
    w, ws = _weights(n, k, 2)
    xs = [torch.randn(m, k, generator=_gen(i), device="cuda").half() for i in range(2)]
    want = [kernels.gemm_rcr_i8(x, w, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(kernels.gemm_rcr_i8(xs[i], w, ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in outs[i])
    graphs = []
    for i, s in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            graphs.append((graph, kernels.gemm_rcr_i8(xs[i], w, ws)))
    for i in range(2):
        xs[i].copy_(torch.randn(m, k, generator=_gen(7 + i), device="cuda"))
    want = [kernels.gemm_rcr_i8(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    for _ in range(10):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, y) for (_, out), y in zip(graphs, want))
