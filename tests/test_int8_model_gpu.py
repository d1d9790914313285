"""The 8-bit operators in a compiled model: the same results, bit for bit, as the eager calls."""
import math

import pytest
import torch

from aitemplate_b200 import kernels
from aitemplate_b200.compiler import compile_model, ops
from aitemplate_b200.frontend import IntVar, Tensor
from aitemplate_b200.testing import detect_target

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weights(n, k, seed):
    g = _gen(seed)
    return (torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8),
            torch.rand(n, generator=g, device="cuda") / (64 * math.sqrt(k)) + 1e-5)


def _out(t, name):
    t._attrs["name"], t._attrs["is_output"] = name, True
    return t


def _param(name, *shape, dtype="float16"):
    return Tensor(list(shape), name=name, dtype=dtype)


@pytest.mark.parametrize("hidden,ffn", [(256, 512), (264, 520), (100, 203)])
def test_feed_forward(tmp_path, hidden, ffn):
    """norm -> 8-bit gated feed-forward -> norm, with a dynamic number of rows, as plain runs and as replayed graphs."""
    rows = IntVar([1, 300], name="rows")
    x, r = (Tensor([rows, hidden], name=n, is_input=True, dtype="bfloat16") for n in ("x", "r"))
    gamma, gate = _param("gamma", hidden, dtype="bfloat16"), _param("gate", hidden, dtype="bfloat16")
    up, ups = _param("up", 2 * ffn, hidden, dtype="int8"), _param("ups", 2 * ffn, dtype="float32")
    down, downs = _param("down", hidden, ffn, dtype="int8"), _param("downs", hidden, dtype="float32")
    total, q, scale = ops.residual_norm("rms", quantize=True)(x, r, gamma=gamma)
    h, hs = ops.quantize_rows("swish", gated=True)(ops.gemm_rcr_i8(dtype="bfloat16")(q, up, ups, scale))
    y = ops.gemm_rcr_i8("add", dtype="bfloat16")(h, down, downs, hs, d0=total)
    last, normed = ops.residual_norm("layer", post_norm="rms", residual_scale=0.5)(y, total, gate)
    module = compile_model([_out(last, "last"), _out(normed, "normed")], detect_target(), str(tmp_path), f"ffn_{hidden}")
    data = dict(zip(("up", "ups"), _weights(2 * ffn, hidden, 1))) | dict(zip(("down", "downs"), _weights(hidden, ffn, 2)))
    for i, name in enumerate(("gamma", "gate")):
        data[name] = (torch.rand(hidden, generator=_gen(i), device="cuda") + 0.5).to(torch.bfloat16)
    module.set_many_constants_with_tensors(data)
    for m in (300, 1, 2, 17, 300, 64):
        xs, rs = (torch.randn(m, hidden, generator=_gen(m + i), device="cuda").to(torch.bfloat16) for i in (0, 1))
        want_total, q8, s8 = kernels.residual_norm(xs, rs, gamma=data["gamma"], norm="rms", quantize=True)
        h8, hs8 = kernels.quantize_rows(kernels.gemm_rcr_i8(q8, data["up"], data["ups"], s8, dtype=torch.bfloat16), "swish", gated=True)
        want_y = kernels.gemm_rcr_i8(h8, data["down"], data["downs"], hs8, d0=want_total, epilogue="add")
        want = kernels.residual_norm(want_y, want_total, data["gate"], post_norm="rms", residual_scale=0.5)
        if hidden % 8 or ffn % 8:
            want = None  # (8-bit rows of a graph lie side by side: the norm takes another kernel, whose sums have another order)
        for graph_mode in (False, True, True):
            outs = {n: torch.full((m, hidden), 7.0, dtype=torch.bfloat16, device="cuda") for n in ("last", "normed")}
            got = module.run_with_tensors({"x": xs, "r": rs}, outs, graph_mode=graph_mode)
            want = want or (got["last"].clone(), got["normed"].clone())
            assert torch.equal(got["last"], want[0]) and torch.equal(got["normed"], want[1])
            assert bool(torch.isfinite(got["normed"].float()).all())
    assert kernels.device_status() == 0
    module.close()


@pytest.mark.parametrize("k,n", [(512, 384), (1000, 70), (77, 33)])
def test_16_bit_rows(tmp_path, k, n):
    """x in 16 bits: quantised in the executor's scratch, or on the way for a few rows. Weights bound at compile time."""
    rows = IntVar([1, 400], name="rows")
    x = Tensor([rows, k], name="x", is_input=True)
    w, ws = _weights(n, k, 3)
    b = torch.randn(n, generator=_gen(4), device="cuda").half()
    y = ops.gemm_rcr_i8("gelu")(x, _param("w", n, k, dtype="int8"), _param("ws", n, dtype="float32"), bias=_param("b", n))
    module = compile_model(_out(y, "y"), detect_target(), str(tmp_path), f"linear_{k}", constants={"w": w.cpu(), "ws": ws.cpu(), "b": b.cpu()})
    for m in (1, 3, 400, 33):
        xs = torch.randn(m, k, generator=_gen(m), device="cuda").half()
        want = kernels.gemm_rcr_i8(xs, w, ws, bias=b, epilogue="gelu")
        for graph_mode in (False, True):
            out = torch.empty((m, n), dtype=torch.float16, device="cuda")
            assert torch.equal(module.run_with_tensors({"x": xs}, {"y": out}, graph_mode=graph_mode)["y"], want)
    module.close()


def test_8_bit_inputs_and_outputs(tmp_path):
    """q and scale as a model's own outputs, and as another one's inputs."""
    x = Tensor([6, 96], name="x", is_input=True)
    q, scale = ops.quantize_rows("relu")(x)
    first = compile_model([_out(q, "q"), _out(scale, "scale")], detect_target(), str(tmp_path), "quantize")
    q_in, s_in = Tensor([6, 96], name="q", dtype="int8", is_input=True), Tensor([6], name="scale", dtype="float32", is_input=True)
    w_in, ws_in = Tensor([40, 96], name="w", dtype="int8", is_input=True), Tensor([40], name="ws", dtype="float32", is_input=True)
    second = compile_model(_out(ops.gemm_rcr_i8()(q_in, w_in, ws_in, s_in), "y"), detect_target(), str(tmp_path), "product")
    xs = torch.randn(6, 96, generator=_gen(0), device="cuda").half()
    outs = {"q": torch.empty(6, 96, dtype=torch.int8, device="cuda"), "scale": torch.empty(6, device="cuda")}
    got = first.run_with_tensors({"x": xs}, outs)
    want = kernels.quantize_rows(xs, "relu")
    assert torch.equal(got["q"], want[0]) and torch.equal(got["scale"], want[1])
    w, ws = _weights(40, 96, 5)
    y = second.run_with_tensors({"q": got["q"], "scale": got["scale"], "w": w, "ws": ws}, {"y": torch.empty(6, 40, dtype=torch.float16, device="cuda")})
    assert torch.equal(y["y"], kernels.gemm_rcr_i8(want[0], w, ws, want[1]))
    with pytest.raises(RuntimeError, match="dtype"):
        second.run_with_tensors({"q": got["q"].half(), "scale": got["scale"], "w": w, "ws": ws}, {"y": torch.empty(6, 40, dtype=torch.float16, device="cuda")})
    first.close(), second.close()


def test_rows_that_do_not_fall_into_parts(tmp_path):
    rows = IntVar([1, 64], name="rows")
    x = Tensor([rows, 64], name="x", is_input=True)
    gate = Tensor([4, 64], name="gate", is_input=True)
    total, y = ops.residual_norm("layer")(x, gate=gate)
    module = compile_model([_out(total, "total"), _out(y, "y")], detect_target(), str(tmp_path), "parts")
    g = torch.randn(4, 64, generator=_gen(1), device="cuda").half()
    for m in (8, 64):
        xs = torch.randn(m, 64, generator=_gen(m), device="cuda").half()
        got = module.run_with_tensors({"x": xs, "gate": g}, {n: torch.empty(m, 64, dtype=torch.float16, device="cuda") for n in ("total", "y")})
        want = kernels.residual_norm(xs, gate=g)
        assert torch.equal(got["total"], want[0]) and torch.equal(got["y"], want[1])
    with pytest.raises(RuntimeError, match="each gate"):
        module.run_with_tensors({"x": xs[:7].contiguous(), "gate": g}, {n: torch.empty(7, 64, dtype=torch.float16, device="cuda") for n in ("total", "y")})
    module.close()
