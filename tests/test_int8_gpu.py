"""gemm_rcr_i8, quantize_rows and residual_norm against their definitions in 64 bits."""
import math

import pytest
import torch

from aitemplate_b200 import kernels

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
STEP32 = 2.0 ** -24  # what rounding to fp32 is off by at most, relative


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int8(g, rows, k, pitch=None):
    store = torch.randint(-128, 128, (rows, pitch or k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return store[:, :k]


def _act64(name, v):
    if name == "relu":
        return v.clamp(min=0)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "fast_gelu":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "sigmoid":
        return torch.sigmoid(v)
    if name == "tanh":
        return torch.tanh(v)
    if name == "swish":
        return v * torch.sigmoid(v)
    if name == "hardswish":
        return v * (v + 3).clamp(0, 6) / 6
    return v


def _act_off(name, v, off):
    """How far an activation in fp32 may be off, of an argument that is `off` off. No slope here passes 1.2. tanh.approx is off by
    2^-11 of its value; exp by its argument's rounding (|v| steps) and 2^-21, and a quotient by 2^-21 more; erf by 2^-22 of 1."""
    own = {"fast_gelu": 0.5 * v.abs() * 2.0 ** -11 + v.abs() * 2.0 ** -20, "tanh": 2.0 ** -11 * torch.ones_like(v),
           "sigmoid": (v.abs() + 16) * STEP32 + 2.0 ** -20, "swish": v.abs() * ((v.abs() + 16) * STEP32 + 2.0 ** -20),
           "gelu": v.abs() * 2.0 ** -20, "hardswish": (v.abs() + 3) * (v.abs() + 3) * 2.0 ** -21}.get(name, 0.0)
    return 1.2 * off + own


def _product64(x, w, xs, ws, bias, d0, d1, epilogue):
    """(result, how far a correct kernel may be off before its last rounding), in 64 bits"""
    u1, b1, b2, u2 = kernels.EPILOGUES[epilogue]
    acc = (x.double() @ w.double().T) * xs.double().reshape(-1, 1) * ws.double()
    off = 4 * STEP32 * acc.abs()  # the sum's conversion, two scales, the addition of the bias
    y = acc
    if bias is not None:
        y = y + bias.double()
        off = off + STEP32 * y.abs()
    y, off = _act64(u1, y), _act_off(u1, y, off)
    for b, d in ((b1, d0), (b2, d1)):
        if b == "add":
            y = y + d.double()
            off = off + STEP32 * y.abs()
        elif b == "mul":
            y = y * d.double()
            off = off * d.double().abs() + STEP32 * y.abs()
    return _act64(u2, y), _act_off(u2, y, off)


def _close(got, want, off, dtype):
    """got = want, `off` off and rounded once to dtype (values under the smallest normal one are rounded to its steps)"""
    half = _half_step(dtype)
    bound = off + half * (want.abs() + off) + torch.finfo(dtype).smallest_normal * half
    away = (got.double() - want).abs()
    assert not torch.isnan(got).any()
    assert bool((away <= bound).all()), f"{float((away / bound).max()):.3f} of the bound"


def _problem(m, n, k, dtype, epilogue, bias, seed, pitch_x=None, pitch_w=None):
    g = _gen(seed)
    x, w = _int8(g, m, k, pitch_x), _int8(g, n, k, pitch_w)
    xs = torch.rand(m, generator=g, device="cuda") / 64 + 0.001
    ws = torch.rand(n, generator=g, device="cuda") / (32 * math.sqrt(k)) + 1e-5
    _, b1, b2, _ = kernels.EPILOGUES[epilogue]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return x, w, ws, xs, rnd(n) if bias else None, rnd(m, n) if b1 else None, rnd(m, n) if b2 else None


def _check_product(m, n, k, dtype, epilogue="", bias=False, seed=0, tile_n=0, pitch_x=None, pitch_w=None):
    x, w, ws, xs, b, d0, d1 = _problem(m, n, k, dtype, epilogue, bias, seed, pitch_x, pitch_w)
    y = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, d0=d0, d1=d1, epilogue=epilogue, dtype=dtype, tile_n=tile_n)
    assert y.shape == (m, n) and y.dtype == dtype
    want, off = _product64(x, w, xs, ws, b, d0, d1, epilogue)
    _close(y, want, off, dtype)
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(128, 128, 128), (1, 128, 256), (16, 256, 512), (256, 256, 256), (300, 520, 336), (7, 64, 16),
                                   (1, 1, 16), (130, 24, 1024), (64, 4096, 768), (1000, 1000, 1008), (5, 10, 32)])
def test_product(m, n, k, dtype):
    _check_product(m, n, k, dtype, bias=True, seed=m + n + k)


@pytest.mark.parametrize("tile_n", [64, 128, 256, 512])
@pytest.mark.parametrize("m,n,k", [(128, 256, 128), (257, 320, 640), (513, 777, 272), (64, 1000, 2048)])
def test_product_by_tile(m, n, k, tile_n):
    a = _check_product(m, n, k, torch.bfloat16, bias=True, seed=m, tile_n=tile_n)
    # sums are exact, and every kernel scales them in the same order
    assert torch.equal(a, _check_product(m, n, k, torch.bfloat16, bias=True, seed=m))


@pytest.mark.parametrize("epilogue", sorted(kernels.EPILOGUES))
@pytest.mark.parametrize("m,n,k,tile_n", [(33, 384, 512, 0), (300, 512, 256, 512), (300, 512, 256, 128), (140, 100, 192, 64),
                                          (140, 515, 192, 256), (260, 515, 192, 512)])
def test_product_epilogues(m, n, k, tile_n, epilogue):
    dtype = DTYPES[len(epilogue) % 2]
    _check_product(m, n, k, dtype, epilogue, bias=epilogue != "mul", seed=len(epilogue), tile_n=tile_n)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 255, 257, 300])
def test_product_few_rows(m):
    for n, k in ((128, 256), (512, 4096), (1027, 1104), (2048, 2048)):
        _check_product(m, n, k, DTYPES[m % 2], bias=m % 3 == 0, epilogue=("", "add", "gelu")[m % 3], seed=m * n)


@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 255, 257, 2041])
def test_product_depths(k):
    """Rows padded to 16 bytes go to the tensor cores, others do not; both give the same result, whatever lies in the padding."""
    pad = (k + 15) // 16 * 16
    for m, n in ((3, 130), (150, 257)):
        x, w, ws, xs, b, _, _ = _problem(m, n, k, torch.float16, "", True, k, pad, pad + 16)
        a = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b)
        c = kernels.gemm_rcr_i8(x.contiguous(), w.contiguous(), ws, xs, bias=b)
        want, off = _product64(x, w, xs, ws, b, None, None, "")
        _close(a, want, off, torch.float16)
        assert torch.equal(a, c)


def test_product_of_the_largest_sums():
    """-128 * -128 over the largest K stays inside 32 bits, on every kernel."""
    k = 131071
    for m, n in ((1, 8), (9, 130), (130, 200)):
        x = torch.full((m, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((n, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w[n // 2] = 127
        xs, ws = torch.full((m,), 2.0 ** -20, device="cuda"), torch.full((n,), 2.0 ** -4, device="cuda")
        want, off = _product64(x, w, xs, ws, None, None, None, "")
        _close(kernels.gemm_rcr_i8(x, w, ws, xs), want, off, torch.float16)


@pytest.mark.parametrize("epilogue", ["", "gelu", "swish", "hardswish"])
def test_product_of_scales_that_are_no_numbers(epilogue):
    """An infinite scale gives infinities, one that is NaN gives NaN, in its row alone and on every kernel."""
    for m, n, k, pad, tile in ((2, 40, 64, 64, 0), (1, 130, 512, 512, 0), (9, 256, 512, 512, 0), (70, 64, 128, 128, 64), (300, 264, 128, 128, 512),
                               (70, 131, 128, 128, 0), (20, 40, 33, 33, 0)):
        x, w, ws, xs, b, _, _ = _problem(m, n, k, torch.float16, "", True, m, pad, pad)
        x.abs_().clamp_(1, 127), w.abs_().clamp_(1, 127)  # (sums above 0)
        clean = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, epilogue=epilogue, tile_n=tile)
        for bad in (math.inf, math.nan):
            xs2 = xs.clone()
            xs2[m // 2] = bad
            y = kernels.gemm_rcr_i8(x, w, ws, xs2, bias=b, epilogue=epilogue, tile_n=tile)
            row = y[m // 2].float()
            assert bool((row == math.inf).all() if bad == math.inf else torch.isnan(row).all()), (m, n, k, bad)
            rest = torch.arange(m, device="cuda") != m // 2
            assert torch.equal(y[rest], clean[rest])


def test_product_leading_dims_and_empty():
    x, w, ws, xs, b, _, _ = _problem(24, 96, 64, torch.float16, "", True, 3)
    y = kernels.gemm_rcr_i8(x, w, ws, xs, bias=b)
    y3 = kernels.gemm_rcr_i8(x.view(2, 3, 4, 64), w, ws, xs.view(2, 3, 4), bias=b)
    assert y3.shape == (2, 3, 4, 96) and torch.equal(y3.view(24, 96), y)
    apart = torch.zeros(24, 3, 64, dtype=torch.int8, device="cuda")
    apart[:, 1] = x
    assert torch.equal(kernels.gemm_rcr_i8(apart[:, 1], w, ws, xs, bias=b), y)
    assert kernels.gemm_rcr_i8(x[:0], w, ws, xs[:0]).shape == (0, 96)
    assert kernels.gemm_rcr_i8(x, w[:0], ws[:0], xs).shape == (24, 0)


def test_product_writes_its_rows_alone():
    """m and n that no tile divides, into the middle of a buffer: what lies around stays as it was."""
    from aitemplate_b200 import _lib

    for m, n, k, tile in ((70, 200, 64, 0), (70, 203, 64, 0), (3, 136, 512, 0), (300, 264, 128, 512), (140, 72, 128, 64)):
        x, w, ws, xs, b, _, _ = _problem(m, n, k, torch.float16, "", True, 5)
        ldc = n + 24
        buf = torch.full((m + 4, ldc), 7.0, dtype=torch.float16, device="cuda")
        out = buf[2:m + 2, 8:8 + n]
        code = _lib.load().b200ait_gemm_rcr_i8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), b.data_ptr(), None, None,
                                               out.data_ptr(), m, n, k, k, k, ldc, n, 0, 1, tile,
                                               torch.cuda.current_stream().cuda_stream)
        _lib.check(code, "b200ait_gemm_rcr_i8")
        assert torch.equal(out, kernels.gemm_rcr_i8(x, w, ws, xs, bias=b))
        out.fill_(7.0)
        assert bool((buf == 7.0).all())


def test_product_random():
    """Sizes, epilogues and types at random, the depth rarely a multiple of anything."""
    import random

    r = random.Random(11)
    for i in range(60):
        m, n, k = (int(math.exp(r.uniform(0, math.log(t)))) for t in (700, 1500, 3000))
        pad = (k + 15) // 16 * 16
        _check_product(m, n, k, r.choice(DTYPES), r.choice(sorted(kernels.EPILOGUES)), r.random() < 0.5, i, r.choice((0, 0, 64, 128, 256, 512)),
                       pad if r.random() < 0.8 else None, pad if r.random() < 0.8 else None)


# ------------------------------------------------------------------------------------------------ quantize_rows
def _quantized64(v):
    most = v.abs().amax(-1, keepdim=True)
    safe = torch.where(most > 0, most, torch.ones_like(most))
    return torch.round(127 * v / safe), (most / 127)[..., 0]


WIDTHS = [1, 2, 7, 8, 9, 16, 31, 100, 256, 257, 768, 1000, 1024, 1032, 1280, 2733, 4096, 5001, 8192, 8200, 16384, 20001, 32768, 32769, 40000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_quantize_rows(n, dtype):
    """Of 16-bit values the result is the definition's to the last bit."""
    for rows in (1, 3, 700 if n <= 1280 else 5):
        x = (torch.randn(rows, n, generator=_gen(n), device="cuda") * torch.logspace(-3, 3, rows, device="cuda")[:, None]).to(dtype)
        q, scale = kernels.quantize_rows(x)
        want, ws = _quantized64(x.double())
        assert q.shape == x.shape and q.dtype == torch.int8 and torch.equal(q.double(), want)
        assert scale.shape == (rows,) and bool(((scale.double() - ws).abs() <= STEP32 * ws).all())
        if n % 16 and rows > 1:
            assert q.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_ties(dtype):
    """Every quotient of two numbers of the type's precision that lands on a half goes to the even side."""
    bits = 8 if dtype == torch.bfloat16 else 11
    top = torch.arange(2 ** (bits - 1), 2 ** bits, device="cuda").double()
    x = torch.cat([top[:, None], top[:, None] / 2, top[:, None] * torch.arange(1, 255, 2, device="cuda") / 256,
                   torch.randint(1, 2 ** bits, (top.numel(), 512), generator=_gen(1), device="cuda").clamp(max=2 ** (bits - 1)).double()], 1)
    x = x.to(dtype)
    q, _ = kernels.quantize_rows(x)
    assert torch.equal(q.double(), _quantized64(x.double())[0])


@pytest.mark.parametrize("n", [5, 64, 4096, 40000])
def test_quantize_rows_extremes(n):
    for dtype in DTYPES:
        info = torch.finfo(dtype)
        rows = torch.zeros(9, n, dtype=dtype, device="cuda")
        rows[1, n - 1] = info.max
        rows[1, 0] = -info.max / 3
        rows[2] = info.tiny * info.eps * 3   # the smallest there are
        rows[2, 0] = -info.tiny * info.eps * 7
        rows[3, n // 2] = math.inf
        rows[4, n // 2] = math.nan
        rows[5, 0], rows[5, n - 1] = -math.inf, math.nan
        rows[6] = -1.0
        rows[7, 1] = info.tiny
        rows[8, 0] = -0.0
        q, scale = kernels.quantize_rows(rows)
        for i in (0, 1, 2, 6, 7, 8):
            want, ws = _quantized64(rows[i].double())
            assert torch.equal(q[i].double(), want), (dtype, i)
            assert abs(float(scale[i]) - float(ws)) <= STEP32 * float(ws) + 2.0 ** -150
        assert float(scale[0]) == 0 and not q[0].any()
        for i in (3, 4, 5):
            assert math.isnan(float(scale[i])) and not q[i].any()
        # a row that could not be quantised shows in the product, and only there
        y = kernels.gemm_rcr_i8(rows, *_weights(24, n, 1), dtype=torch.bfloat16)
        bad = torch.isnan(y).any(1)
        assert bad.tolist() == [False, False, False, True, True, True, False, False, False]
        assert bool(torch.isnan(y[bad]).all())


def _weights(n, k, seed):
    g = _gen(seed)
    return _int8(g, n, k, (k + 15) // 16 * 16), torch.rand(n, generator=g, device="cuda") / (32 * math.sqrt(k)) + 1e-5


def _near_quantized(q, scale, v, off):
    """v is known to `off`: q * scale is then half a step from it at most (and as far again as v may be off)"""
    most = v.abs().amax(-1)
    assert bool(((scale.double() * 127 - most).abs() <= off.amax(-1) + 2 * STEP32 * most + 1e-300).all())
    away = (q.double() * scale.double()[..., None] - v).abs()
    assert bool((away <= scale.double()[..., None] * (0.5 + 1e-4) + 2 * off + 1e-300).all())
    assert int(q.abs().max()) <= 127
    want = torch.round(127 * v / most[..., None].clamp(min=1e-300))
    assert float((q.double() != want).double().mean()) < 0.02 and float((q.double() - want).abs().max()) <= 1


@pytest.mark.parametrize("activation", sorted(kernels.UNARY))
@pytest.mark.parametrize("n", [8, 33, 768, 2733, 4096, 33000])
def test_quantize_gated_rows(n, activation):
    for rows, dtype, gated in ((1, torch.float16, True), (9, torch.bfloat16, True), (300, torch.float16, False)):
        if n > 5000 and rows > 10:
            continue
        x = torch.randn(rows, n * (2 if gated else 1), generator=_gen(n), device="cuda").to(dtype)
        q, scale = kernels.quantize_rows(x, activation, gated=gated)
        g = x[:, :n].double()
        v, off = _act64(activation, g), _act_off(activation, g, STEP32 * g.abs())
        if gated:
            u = x[:, n:].double()
            v, off = v * u, (off + STEP32 * v.abs()) * u.abs()
        _near_quantized(q, scale, v, off)


def test_quantize_rows_apart():
    x = torch.randn(40, 3, 200, generator=_gen(4), device="cuda").to(torch.bfloat16)
    a, sa = kernels.quantize_rows(x[:, 1])
    b, sb = kernels.quantize_rows(x[:, 1].contiguous())
    assert torch.equal(a, b) and torch.equal(sa, sb)
    c, sc = kernels.quantize_rows(x)
    assert c.shape == (40, 3, 200) and torch.equal(c[:, 1], b) and torch.equal(sc[:, 1], sb)
    odd = torch.randn(40, 401, generator=_gen(5), device="cuda").to(torch.float16)[:, 1:]  # rows off 16 bytes
    d, sd = kernels.quantize_rows(odd)
    assert torch.equal(d.double(), _quantized64(odd.double())[0])
    empty, se = kernels.quantize_rows(x[:0])
    assert empty.shape == (0, 3, 200) and se.shape == (0, 3)


# ------------------------------------------------------------------------------------------------ residual_norm
def _norm64(kind, v, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def _spread(t, rows):
    """a vector per part of the rows, for every row"""
    t = t.double()
    return t if t.dim() == 1 else t.repeat_interleave(rows // t.shape[0], 0)


def _residual_norm64(x, o):
    """((total, off), (y, off)) in 64 bits; `off`: how far fp32 may be from it. A sum of n terms in a tree of threads, each of 32
    terms at most and then in pairs, is off by 64 steps of the sum of magnitudes; a norm's statistics then move a value by as many
    steps of the row's largest one over its deviation, and the values by a few steps of their own."""
    p, off, n = x.double(), torch.zeros_like(x.double()), x.shape[-1]

    def norm(kind, v, off):
        away = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        sd = torch.sqrt((away * away).mean(-1, keepdim=True) + o["eps"])
        y = away / sd
        worst = 64 * STEP32 * v.abs().mean(-1, keepdim=True) + off.amax(-1, keepdim=True)  # of the mean, and of any value
        return y, 2 * (worst + off + 2 * STEP32 * v.abs()) / sd + y.abs() * (2 * worst / sd + 72 * STEP32)

    if o["post_norm"]:
        p, off = norm(o["post_norm"], p, off)
        if o["post_gamma"] is not None:
            p, off = p * o["post_gamma"].double(), off * o["post_gamma"].double().abs()
        if o["post_beta"] is not None:
            p = p + o["post_beta"].double()
        off = off + 2 * STEP32 * p.abs()
    if o["gate"] is not None:
        gate = _spread(o["gate"], x.shape[0])
        p, off = p * gate, off * gate.abs() + STEP32 * (p * gate).abs()
    total = p if o["residual"] is None else p + o["residual_scale"] * o["residual"].double()
    off = off + 2 * STEP32 * (total.abs() + p.abs())
    y, off_y = norm(o["norm"], total, off)
    if o["gamma"] is not None:
        g = _spread(o["gamma"], x.shape[0])
        y, off_y = y * g, off_y * g.abs()
    if o["beta"] is not None:
        y = y + _spread(o["beta"], x.shape[0])
    return (total, off), (y, off_y + 2 * STEP32 * y.abs())


def _norm_operands(rows, n, dtype, seed, parts=1, post="rms", norm="layer", leave_out=()):
    g = _gen(seed)
    rnd = lambda *s, a=1.0, b=0.0: (torch.randn(*s, generator=g, device="cuda") * a + b).to(dtype)  # noqa: E731
    x = rnd(rows, n, a=2.0, b=0.5)
    o = {"residual": rnd(rows, n, a=3.0), "gate": rnd(parts, n), "post_gamma": rnd(n, a=0.2, b=1.0) if post else None,
         "post_beta": rnd(n, a=0.2) if post else None, "gamma": rnd(parts, n, a=0.2, b=1.0), "beta": rnd(n, a=0.2), "post_norm": post,
         "norm": norm, "residual_scale": 0.75, "eps": 1e-5}
    if parts == 1:
        o["gate"], o["gamma"] = o["gate"][0], o["gamma"][0]
    for name in leave_out:
        o[name] = None
    return x, o


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_residual_norm(n, dtype):
    kinds = [(None, "layer"), ("rms", "rms"), ("layer", "rms"), ("layer", "layer")]
    for i, (rows, parts) in enumerate(((1, 1), (6, 3), (700 if n <= 1280 else 8, 4))):
        post, norm = kinds[(n + i) % 4]
        if n == 1:
            norm, post = "rms", None  # (the layer norm of one value is 0 over 0)
        x, o = _norm_operands(rows, n, dtype, n + i, parts, post, norm)
        (total, off_t), (want, off_y) = _residual_norm64(x, o)
        s, y = kernels.residual_norm(x, **o)
        assert s.dtype == y.dtype == dtype and s.shape == y.shape == x.shape
        _close(s, total, off_t, dtype)
        _close(y, want, off_y, dtype)
        s8, q, scale = kernels.residual_norm(x, quantize=True, **o)
        assert torch.equal(s8, s)
        _near_quantized(q, scale, want, off_y)


# many rows: a width for every number of threads and of 8-element units a thread, of rows that start on 16 bytes and of others
MANY = [8 * u for u in (20, 40, 72, 104, 136, 168, 200, 264, 328, 400, 520, 648, 800, 1032, 1300, 1544, 2056, 2568, 3080)]
MANY += [200 - 7, 505, 761, 1001, 1529, 2041, 2901, 4001, 6001, 8001, 12001, 16001, 24001]


@pytest.mark.parametrize("n", MANY)
def test_many_rows(n):
    dtype = DTYPES[n // 8 % 2]
    x = torch.randn(601, n, generator=_gen(n), device="cuda").to(dtype)
    q, scale = kernels.quantize_rows(x)
    want, ws = _quantized64(x.double())
    assert torch.equal(q.double(), want)
    assert bool(((scale.double() - ws.flatten()).abs() <= STEP32 * ws.flatten()).all())
    x, o = _norm_operands(304, n, dtype, n, 4, (None, "rms", "layer")[n % 3], ("layer", "rms")[n % 2])
    (total, off_t), (want, off_y) = _residual_norm64(x, o)
    s, y = kernels.residual_norm(x, **o)
    _close(s, total, off_t, dtype)
    _close(y, want, off_y, dtype)
    s8, q, scale = kernels.residual_norm(x, quantize=True, **o)
    assert torch.equal(s8, s)
    _near_quantized(q, scale, want, off_y)


@pytest.mark.parametrize("leave_out", [("residual",), ("gate",), ("gamma", "beta"), ("post_gamma",), ("post_beta", "beta"),
                                       ("residual", "gate", "post_gamma", "post_beta", "gamma", "beta")])
@pytest.mark.parametrize("n", [768, 1001, 2048])
def test_residual_norm_left_out(n, leave_out):
    x, o = _norm_operands(50, n, torch.float16, n, 1, "layer", "rms", leave_out)
    (total, off_t), (want, off_y) = _residual_norm64(x, o)
    s, y = kernels.residual_norm(x, **o)
    _close(s, total, off_t, torch.float16)
    _close(y, want, off_y, torch.float16)


def test_residual_norm_rows_stand_alone():
    """Rows of zeros, and rows with an infinity or a NaN, among others: each row's result is its own."""
    for n in (64, 999, 4096, 33000):
        x, o = _norm_operands(6, n, torch.bfloat16, n, 1, "rms", "layer")
        clean = kernels.residual_norm(x, quantize=True, **o)
        x[1], x[3, n // 2], x[4, 0] = 0, math.nan, math.inf
        s, q, scale = kernels.residual_norm(x, quantize=True, **o)
        for row in (0, 2, 5):
            assert all(torch.equal(a[row], b[row]) for a, b in zip(clean, (s, q, scale)))
        (total, off_t), (want, off_y) = _residual_norm64(x[1:2], {**o, "residual": o["residual"][1:2]})
        _close(s[1:2], total, off_t, torch.bfloat16)
        _near_quantized(q[1:2], scale[1:2], want, off_y)
        assert math.isnan(float(scale[3])) and math.isnan(float(scale[4])) and not q[3].any() and not q[4].any()
        assert bool(torch.isnan(kernels.residual_norm(x, **o)[1][3]).all())


def _at(t, elements):
    """a contiguous copy of t that starts `elements` elements after a 16-byte boundary"""
    store = torch.full((t.numel() + elements + 8,), 7.0, dtype=t.dtype, device=t.device)
    store[elements:elements + t.numel()] = t.reshape(-1)
    return store[elements:elements + t.numel()].view(t.shape)


@pytest.mark.parametrize("n", [8, 9, 31, 264, 1001, 1280, 4100])
@pytest.mark.parametrize("place", [0, 1, 4, 7])
def test_rows_anywhere_in_memory(n, place):
    """The result does not depend on where the operands lie, alike or each at a place of its own."""
    rows = 21
    x, o = _norm_operands(rows, n, torch.bfloat16, n, 3, "layer", "rms")
    want = kernels.residual_norm(x, quantize=True, **o), kernels.residual_norm(x, **o)
    for moved in (("residual",), ("gamma",), ("gate", "post_beta"), ("residual", "gate", "gamma", "beta", "post_gamma", "post_beta")):
        p = {k: _at(v, (place + i) % 8) if k in moved else v for i, (k, v) in enumerate(o.items())}
        got = kernels.residual_norm(_at(x, place), quantize=True, **p), kernels.residual_norm(_at(x, place), **p)
        for a, b in zip(want, got):
            for c, d in zip(a, b):
                if c.dtype == torch.int8:
                    assert float((c != d).double().mean()) < 0.01 and int((c.int() - d.int()).abs().max()) <= 1
                else:  # (sums in another order)
                    assert torch.allclose(c.float(), d.float(), rtol=2.0 ** -7, atol=1e-5)
    v = x[:, :n // 2 * 2]
    for gated in (False, True):
        if gated and n < 16:
            continue
        a = kernels.quantize_rows(v.contiguous(), "relu", gated=gated)
        b = kernels.quantize_rows(_at(v.contiguous(), place), "relu", gated=gated)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_results_stay_in_their_rows():
    """What lies between and around the rows of q, total and y stays as it was, wherever the rows end."""
    from aitemplate_b200 import _lib

    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for n in (1, 7, 8, 9, 15, 100, 257, 1003, 2049, 4104):
        pitch = (n + 15) // 16 * 16 + 16
        x = torch.randn(5, n, generator=_gen(n), device="cuda").to(torch.float16)
        q = torch.full((7, pitch), 99, dtype=torch.int8, device="cuda")
        scale = torch.full((7,), 5.0, device="cuda")
        _lib.check(lib.b200ait_quantize_rows(q[1:].data_ptr(), scale[1:].data_ptr(), x.data_ptr(), 5, n, n, pitch, 0, 0, 1, stream), "")
        want, ws = kernels.quantize_rows(x)
        assert torch.equal(q[1:6, :n], want) and torch.equal(scale[1:6], ws)
        assert bool((q[1:6, n:] == 99).all()) and bool((q[[0, 6]] == 99).all()) and scale[0] == 5 and scale[6] == 5
        total, y = (torch.full((5 * n + 32,), 99.0, dtype=torch.float16, device="cuda") for _ in range(2))
        for lead in (8, 3):
            total.fill_(99), y.fill_(99), q.fill_(99), scale.fill_(5)
            a, b = _at(x, lead), _at(x, lead)
            _lib.check(lib.b200ait_residual_norm(total[lead:].data_ptr(), y[lead:].data_ptr(), None, a.data_ptr(), b.data_ptr(), None, None,
                                                 None, None, None, 5, n, 1, 1, 1, 0, 0, 2, 1.0, 1e-5, 1, stream), "")
            for t in (total, y):
                assert bool((t[:lead] == 99).all()) and bool((t[lead + 5 * n:] == 99).all())
            assert torch.equal(total[lead:lead + 5 * n].view(5, n), x + x)
            _lib.check(lib.b200ait_residual_norm(None, q[1:].data_ptr(), scale[1:].data_ptr(), a.data_ptr(), b.data_ptr(), None, None,
                                                 None, None, None, 5, n, 1, 1, 1, pitch, 0, 2, 1.0, 1e-5, 1, stream), "")
            assert bool((q[1:6, n:] == 99).all()) and bool((q[[0, 6]] == 99).all()) and scale[0] == 5 and scale[6] == 5
            assert bool((q[1:6, :n].abs().amax(1) == 127).all())


def test_residual_norm_in_place():
    """total may be written over the residual, or over x."""
    from aitemplate_b200 import _lib

    for n in (1000, 1001, 40000):
        x, o = _norm_operands(9, n, torch.float16, n, 1, None, "layer")
        want = kernels.residual_norm(x, **o)
        for over in ("residual", "x"):
            a, r = x.clone(), o["residual"].clone()
            y = torch.empty_like(x)
            _lib.check(_lib.load().b200ait_residual_norm(
                (r if over == "residual" else a).data_ptr(), y.data_ptr(), None, a.data_ptr(), r.data_ptr(), o["gate"].data_ptr(), None, None,
                o["gamma"].data_ptr(), o["beta"].data_ptr(), 9, n, 1, 1, 1, 0, 0, 1, 0.75, 1e-5, 1, torch.cuda.current_stream().cuda_stream), "")
            assert torch.equal(r if over == "residual" else a, want[0]) and torch.equal(y, want[1])


def test_residual_norm_leading_dims_and_empty():
    x, o = _norm_operands(24, 256, torch.float16, 2, 2, None, "rms")
    s, y = kernels.residual_norm(x, **o)
    s3, y3 = kernels.residual_norm(x.view(2, 12, 256), **{**o, "residual": o["residual"].view(2, 12, 256)})
    assert torch.equal(s3.view(24, 256), s) and torch.equal(y3.view(24, 256), y)
    s0, q0, c0 = kernels.residual_norm(x[:0], residual=o["residual"][:0], gate=o["gate"], quantize=True)
    assert s0.shape == (0, 256) and q0.shape == (0, 256) and c0.shape == (0,)


# ------------------------------------------------------------------------------------------------ together
def _feed_forward(x, residual, gamma, w_up, w_down, dtype):
    total, q, scale = kernels.residual_norm(x, residual, gamma=gamma, norm="rms", quantize=True)
    up = kernels.gemm_rcr_i8(q, w_up[0], w_up[1], scale, dtype=dtype)
    h, hs = kernels.quantize_rows(up, "swish", gated=True)
    return total, kernels.gemm_rcr_i8(h, w_down[0], w_down[1], hs, d0=total, epilogue="add", dtype=dtype)


@pytest.mark.parametrize("rows,n,ffn", [(1, 512, 1000), (5, 768, 2040), (300, 256, 520)])
def test_a_block_of_them(rows, n, ffn):
    """The norm, the gated feed-forward in 8 bits and the residual, as a program calls them one after the other; each step against 64 bits
    from what the step before handed on."""
    dtype = torch.bfloat16
    g = _gen(rows)
    x, residual = (torch.randn(rows, n, generator=g, device="cuda").to(dtype) for _ in range(2))
    gamma = (torch.rand(n, generator=g, device="cuda") + 0.5).to(dtype)
    w_up, w_down = _weights(2 * ffn, n, 7), _weights(n, ffn, 8)
    total, y = _feed_forward(x, residual, gamma, w_up, w_down, dtype)
    _, q, scale = kernels.residual_norm(x, residual, gamma=gamma, norm="rms", quantize=True)
    up = kernels.gemm_rcr_i8(q, w_up[0], w_up[1], scale, dtype=dtype)
    want, off = _product64(q, w_up[0], scale, w_up[1], None, None, None, "")
    _close(up, want, off, dtype)
    h, hs = kernels.quantize_rows(up, "swish", gated=True)
    want, off = _product64(h, w_down[0], hs, w_down[1], None, total, None, "add")
    _close(y, want, off, dtype)


def test_captured_and_on_another_stream():
    dtype, rows, n, ffn = torch.bfloat16, 37, 384, 520
    g = _gen(3)
    x, residual = (torch.randn(rows, n, generator=g, device="cuda").to(dtype) for _ in range(2))
    gamma = (torch.rand(n, generator=g, device="cuda") + 0.5).to(dtype)
    w_up, w_down = _weights(2 * ffn, n, 7), _weights(n, ffn, 8)
    total, y = _feed_forward(x, residual, gamma, w_up, w_down, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t2, y2 = _feed_forward(x, residual, gamma, w_up, w_down, dtype)
    torch.cuda.synchronize()
    assert torch.equal(total, t2) and torch.equal(y, y2)
    graphs = []
    for _ in range(2):  # two graphs that may run one inside the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _feed_forward(x, residual, gamma, w_up, w_down, dtype)
        graphs.append((graph, out))
    other = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    want = _feed_forward(other, residual, gamma, w_up, w_down, dtype)
    x.copy_(other)
    for graph, _ in graphs:
        graph.replay()
    for _, out in graphs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 40, 200])
@pytest.mark.parametrize("k", [1, 8, 300, 512, 1023, 1024, 2041, 4096, 10000])
def test_16_bit_rows_are_quantised_on_the_way(m, k):
    """In one call or two, by the product's own kernel or into scratch: the same result."""
    for dtype, out in ((torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.bfloat16)):
        x = torch.randn(m, k, generator=_gen(m), device="cuda").to(dtype)
        x[m // 2, :k // 2] *= 40
        w, ws = _weights(139, k, 2)
        b, d0 = (torch.randn(*s, generator=_gen(k), device="cuda").to(out) for s in ((139,), (m, 139)))
        q, scale = kernels.quantize_rows(x)
        want = kernels.gemm_rcr_i8(q, w, ws, scale, bias=b, d0=d0, epilogue="add", dtype=out)
        ref, off = _product64(q, w, scale, ws, b, d0, None, "add")
        _close(want, ref, off, out)
        for form in (x, _at(x, 3), torch.cat([x, x, x], 1)[:, k:2 * k]):  # rows on and off 16 bytes, and apart
            assert torch.equal(kernels.gemm_rcr_i8(form, w, ws, bias=b, d0=d0, epilogue="add", dtype=out), want)
        assert torch.equal(kernels.gemm_rcr_i8(x, w.contiguous(), ws, bias=b, d0=d0, epilogue="add", dtype=out), want)
    x[0, 0] = math.inf
    y = kernels.gemm_rcr_i8(x, w, ws)
    assert bool(torch.isnan(y[0]).all()) and not torch.isnan(y[1:]).any()


def test_a_few_rows_of_any_place_and_shape():
    """One to four rows against many, few and no whole turns of columns, W with rows apart and its last row at the end of its memory."""
    for m in (1, 2, 3, 4):
        for n, k in ((1, 64), (2, 5000), (37, 512), (148, 513), (593, 1024), (3001, 1040), (4097, 528), (600, 2064), (9000, 256), (300, 20000)):
            _check_product(m, n, k, DTYPES[n % 2], ("", "add", "mul_add", "gelu")[(m + n) % 4], True, n, pitch_w=(k + 31) // 16 * 16)


def test_the_native_path_and_the_python_code_agree(monkeypatch):
    from aitemplate_b200 import _lib

    class Absent:
        def __getattr__(self, name):
            return lambda *args: None

    class Recorder:
        def __init__(self):
            self.module, self.served = _lib.load_calls(), []

        def __getattr__(self, name):
            def call(*args):
                y = getattr(self.module, name)(*args)
                self.served.append(y is not None)
                return y
            return call

    x, w, ws, xs, b, d0, _ = _problem(6, 40, 72, torch.float16, "add", True, 1, 80, 96)
    h = torch.randn(2, 3, 72, generator=_gen(1), device="cuda").to(torch.bfloat16)
    n, o = _norm_operands(6, 72, torch.float16, 1, 3, "rms", "layer")
    calls = [
        lambda: kernels.gemm_rcr_i8(x, w, ws, xs, bias=b, d0=d0, epilogue="add"), lambda: kernels.gemm_rcr_i8(x, w, ws, xs),
        lambda: kernels.gemm_rcr_i8(x, w, ws, xs, dtype=torch.bfloat16, tile_n=64), lambda: kernels.gemm_rcr_i8(h, w, ws),
        lambda: kernels.gemm_rcr_i8(h, w, ws, dtype=torch.float16), lambda: kernels.gemm_rcr_i8(h[0, :1], w, ws, bias=b.bfloat16()),
        lambda: kernels.gemm_rcr_i8(h[:, 1], w, ws), lambda: kernels.quantize_rows(h), lambda: kernels.quantize_rows(h[:, 1], "swish", True),
        lambda: kernels.quantize_rows(torch.nn.Parameter(h[0])), lambda: kernels.residual_norm(n, **o),
        lambda: kernels.residual_norm(n, quantize=True, **o), lambda: kernels.residual_norm(h, norm="rms"),
    ]
    for call in calls:
        with monkeypatch.context() as c:
            recorder = Recorder()
            c.setattr(kernels, "_calls", recorder)
            native = call()
            assert recorder.served == [True]
        with monkeypatch.context() as c:
            c.setattr(kernels, "_calls", Absent())
            python = call()
        for p, q in zip(*((r,) if torch.is_tensor(r) else r for r in (native, python))):
            assert p.shape == q.shape and p.dtype == q.dtype and p.stride() == q.stride() and torch.equal(p, q)


def test_another_device_is_refused(monkeypatch):
    x, w, ws, xs, *_ = _problem(6, 32, 64, torch.float16, "", False, 1)

    class Absent:
        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(kernels, "_calls", Absent())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: kernels.gemm_rcr_i8(x, w, ws, xs), lambda: kernels.quantize_rows(xs), lambda: kernels.residual_norm(xs)):
        with pytest.raises(ValueError, match="the current device is cuda:1"):
            call()


def test_one_dimension():
    x, w, ws, xs, b, _, _ = _problem(1, 40, 64, torch.float16, "", True, 1)
    assert torch.equal(kernels.gemm_rcr_i8(x[0], w, ws, xs[0], bias=b), kernels.gemm_rcr_i8(x, w, ws, xs, bias=b)[0])
    v = torch.randn(70, generator=_gen(1), device="cuda").half()
    (q, s), (q2, s2) = kernels.quantize_rows(v), kernels.quantize_rows(v[None])
    assert q.shape == (70,) and s.shape == () and torch.equal(q, q2[0]) and torch.equal(s, s2[0])
    assert torch.equal(kernels.residual_norm(v)[1], kernels.residual_norm(v[None])[1][0])


def test_refusals():
    x, w, ws, xs, b, d0, _ = _problem(6, 32, 64, torch.float16, "add", True, 1)
    call = kernels.gemm_rcr_i8
    for wrong, said in (
        (lambda: call(x, w, ws), "needs x_scale"), (lambda: call(x.half(), w, ws, xs), "goes with an int8"),
        (lambda: call(x, w[:, :48], ws, xs), "K mismatch"), (lambda: call(x, w, ws[:8], xs), "w_scale"),
        (lambda: call(x, w, ws, xs.half()), "x_scale"), (lambda: call(x, w.half(), ws, xs), "w must be int8"),
        (lambda: call(x, w, ws, xs, epilogue="add"), "needs d0"), (lambda: call(x, w, ws, xs, d0=d0), "takes no d0"),
        (lambda: call(x, w, ws, xs, bias=b.bfloat16(), dtype=torch.float16), "bias must be"),
        (lambda: call(x, w, ws, xs, epilogue="square"), "unknown epilogue"), (lambda: call(x, w, ws, xs, dtype=torch.float32), "unsupported dtype"),
        (lambda: call(x[:, ::2], w[:, :32], ws, xs), "side by side"), (lambda: call(x[:, :0], w[:, :0], ws, xs), "K is 0"),
        (lambda: call(x, w.cpu(), ws, xs), "CUDA tensor"), (lambda: call(x.expand(2, 6, 64), w, ws, xs.expand(2, 6).contiguous()), "one distance"),
        (lambda: kernels.quantize_rows(x), "unsupported dtype"), (lambda: kernels.quantize_rows(b, gated=True, activation="elu"), "unknown activation"),
        (lambda: kernels.quantize_rows(b[:7], gated=True), "two halves"), (lambda: kernels.quantize_rows(b[:0]), "no columns"),
        (lambda: kernels.residual_norm(d0, d0[:3]), "does not fit"), (lambda: kernels.residual_norm(d0, gate=d0[:4]), "does not fit"),
        (lambda: kernels.residual_norm(d0, norm="batch"), "a norm is"), (lambda: kernels.residual_norm(d0, post_gamma=b), "need a post_norm"),
        (lambda: kernels.residual_norm(d0, d0.bfloat16()), "must be a contiguous"), (lambda: kernels.residual_norm(x, x), "unsupported dtype"),
    ):
        with pytest.raises(ValueError, match=said):
            wrong()
    with pytest.raises(RuntimeError, match="131071"):
        call(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), torch.zeros(8, 131072, dtype=torch.int8, device="cuda"), ws[:8], xs[:1])
    with pytest.raises(RuntimeError, match="tile_n"):
        call(x, w, ws, xs, tile_n=96)
