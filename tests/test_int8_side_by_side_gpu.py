"""Widths that are no multiple of 8 in a compiled model, where 8-bit rows lie side by side: the same, bit for bit, as the C entries at that pitch, whose
steps are checked against 64 bits one by one."""
import pytest
import torch

from aitemplate_b200 import _lib, kernels
from aitemplate_b200.compiler import compile_model, ops
from aitemplate_b200.frontend import IntVar, Tensor
from aitemplate_b200.testing import detect_target
from test_int8_gpu import _act64, _act_off, _close, _gen, _near_quantized, _product64, _residual_norm64, STEP32
from test_int8_model_gpu import _out, _param, _weights

pytestmark = pytest.mark.gpu
BF16 = 6


def _p(t):
    return None if t is None else t.data_ptr()


def _norm_to_8(x, r, gamma):
    m, n = x.shape
    total, q, scale = torch.empty_like(x), torch.empty(m, n, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    code = _lib.load().b200ait_residual_norm(_p(total), _p(q), _p(scale), _p(x), _p(r), None, None, None, _p(gamma), None, m, n, 1, 1, 1, n, 0, 2, 1.0,
                                             1e-5, BF16, torch.cuda.current_stream().cuda_stream)
    _lib.check(code, "b200ait_residual_norm")
    return total, q, scale


def _gated_to_8(x):
    m, n = x.shape[0], x.shape[1] // 2
    q, scale = torch.empty(m, n, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    code = _lib.load().b200ait_quantize_rows(_p(q), _p(scale), _p(x), m, n, 2 * n, n, kernels.UNARY["swish"], 1, BF16,
                                             torch.cuda.current_stream().cuda_stream)
    _lib.check(code, "b200ait_quantize_rows")
    return q, scale


@pytest.mark.parametrize("hidden,ffn", [(100, 203), (77, 129), (136, 203)])
def test_feed_forward_of_odd_widths(tmp_path, hidden, ffn):
    rows = IntVar([1, 300], name="rows")
    x, r = (Tensor([rows, hidden], name=n, is_input=True, dtype="bfloat16") for n in ("x", "r"))
    gamma = _param("gamma", hidden, dtype="bfloat16")
    up, ups = _param("up", 2 * ffn, hidden, dtype="int8"), _param("ups", 2 * ffn, dtype="float32")
    down, downs = _param("down", hidden, ffn, dtype="int8"), _param("downs", hidden, dtype="float32")
    total, q, scale = ops.residual_norm("rms", quantize=True)(x, r, gamma=gamma)
    h, hs = ops.quantize_rows("swish", gated=True)(ops.gemm_rcr_i8(dtype="bfloat16")(q, up, ups, scale))
    y = ops.gemm_rcr_i8("add", dtype="bfloat16")(h, down, downs, hs, d0=total)
    module = compile_model([_out(total, "total"), _out(y, "y")], detect_target(), str(tmp_path), f"side_{hidden}_{ffn}")
    data = dict(zip(("up", "ups"), _weights(2 * ffn, hidden, 1))) | dict(zip(("down", "downs"), _weights(hidden, ffn, 2)))
    data["gamma"] = (torch.rand(hidden, generator=_gen(0), device="cuda") + 0.5).to(torch.bfloat16)
    module.set_many_constants_with_tensors(data)
    for m in (300, 1, 2, 17, 64):
        xs, rs = (torch.randn(m, hidden, generator=_gen(m + i), device="cuda").to(torch.bfloat16) for i in (0, 1))
        o = {"residual": rs, "gate": None, "post_gamma": None, "post_beta": None, "gamma": data["gamma"], "beta": None, "post_norm": None, "norm": "rms",
             "residual_scale": 1.0, "eps": 1e-5}
        (total64, off_t), (normed64, off_n) = _residual_norm64(xs, o)
        total, q, scale = _norm_to_8(xs, rs, data["gamma"])
        _close(total, total64, off_t, torch.bfloat16)
        _near_quantized(q, scale, normed64, off_n)
        up_y = kernels.gemm_rcr_i8(q, data["up"], data["ups"], scale, dtype=torch.bfloat16)
        _close(up_y, *_product64(q, data["up"], scale, data["ups"], None, None, None, ""), torch.bfloat16)
        h, hs = _gated_to_8(up_y)
        g, u = up_y[:, :ffn].double(), up_y[:, ffn:].double()
        v, off = _act64("swish", g), _act_off("swish", g, STEP32 * g.abs())
        _near_quantized(h, hs, v * u, (off + STEP32 * v.abs()) * u.abs())
        want = kernels.gemm_rcr_i8(h, data["down"], data["downs"], hs, d0=total, epilogue="add")
        _close(want, *_product64(h, data["down"], hs, data["downs"], None, total, None, "add"), torch.bfloat16)
        for graph_mode in (False, True, True):
            outs = {n: torch.full((m, hidden), 7.0, dtype=torch.bfloat16, device="cuda") for n in ("total", "y")}
            got = module.run_with_tensors({"x": xs, "r": rs}, outs, graph_mode=graph_mode)
            assert torch.equal(got["total"], total) and torch.equal(got["y"], want)
    assert kernels.device_status() == 0
    module.close()
