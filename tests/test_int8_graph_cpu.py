"""Graph nodes of the 8-bit operators: shapes, types, refusals and the plan they lower to."""
import pytest

from aitemplate_b200.compiler import ops
from aitemplate_b200.compiler.compiler import _assign_storage, _lower_to_plan
from aitemplate_b200.compiler.dtype import dtype_enum_to_str, dtype_str_to_enum, get_dtype_size
from aitemplate_b200.compiler.transform import mark_param_tensor, memory_planning, name_graph, toposort
from aitemplate_b200.frontend import IntVar, Tensor


def _t(name, *shape, dtype="float16", is_input=True):
    return Tensor(list(shape), name=name, dtype=dtype, is_input=is_input)


def _plan(*outputs):
    for i, y in enumerate(outputs):
        y._attrs["name"], y._attrs["is_output"] = f"out_{i}", True
    graph = toposort(list(outputs))
    mark_param_tensor(graph)
    name_graph(graph)
    copies = _assign_storage(graph, list(outputs))
    blob, constants = memory_planning(graph)
    return _lower_to_plan(graph, list(outputs), "t", blob, constants, copies, None, {}).splitlines()


def test_int8_is_a_type_of_its_own():
    assert dtype_str_to_enum("int8") == 7 and dtype_enum_to_str(7) == "int8" and get_dtype_size("int8") == 1
    assert _t("x", 3, 5, dtype="int8").size_bytes() == 15


def test_shapes_and_types():
    m = IntVar([1, 64], name="m")
    x = _t("x", m, 10, 96, dtype="bfloat16")
    q, scale = ops.quantize_rows("swish", gated=True)(x)
    assert [d.upper_bound() for d in q._attrs["shape"]] == [64, 10, 48] and q.dtype() == "int8"
    assert [d.upper_bound() for d in scale._attrs["shape"]] == [64, 10] and scale.dtype() == "float32"
    w, ws = _t("w", 32, 48, dtype="int8", is_input=False), _t("ws", 32, dtype="float32", is_input=False)
    y = ops.gemm_rcr_i8("relu", dtype="bfloat16")(q, w, ws, scale)
    assert [d.upper_bound() for d in y._attrs["shape"]] == [64, 10, 32] and y.dtype() == "bfloat16"
    total, y8, s8 = ops.residual_norm("rms", quantize=True)(y, _t("r", m, 10, 32, dtype="bfloat16"))
    assert total.dtype() == "bfloat16" and y8.dtype() == "int8" and s8.dtype() == "float32"
    assert ops.gemm_rcr_i8()(q, w, ws, scale).dtype() == "float16"
    assert ops.gemm_rcr_i8()(_t("h", m, 48, dtype="bfloat16"), w, ws).dtype() == "bfloat16"


def test_lowering():
    m = IntVar([1, 64], name="m")
    x, r = _t("x", m, 64), _t("r", m, 64)
    gamma = _t("gamma", 64, is_input=False)
    w, ws = _t("w", 128, 64, dtype="int8", is_input=False), _t("ws", 128, dtype="float32", is_input=False)
    total, q, scale = ops.residual_norm("layer", residual_scale=0.5, quantize=True)(x, r, gamma=gamma)
    h, hs = ops.quantize_rows("gelu", gated=True)(ops.gemm_rcr_i8()(q, w, ws, scale))
    w2, ws2 = _t("w2", 64, 64, dtype="int8", is_input=False), _t("ws2", 64, dtype="float32", is_input=False)
    lines = _plan(ops.gemm_rcr_i8("add")(h, w2, ws2, hs, d0=total))
    found = [l.split() for l in lines if l.startswith("op ")]
    assert [l[1] for l in found] == ["residual_norm", "gemm_rcr_i8", "quantize_rows", "gemm_rcr_i8"]
    kinds = {int(i): l.split() for i, l in enumerate(l for l in lines if l.startswith("tensor "))}
    assert {kinds[int(i)][2] for i in found[0][13:15]} <= {"1", "7", "2"}
    # residual_norm: no norm after the block, layer, 8 bits, the sum has a reader
    assert " 4 0 1 1 1 2 0.5 1e-05" in " ".join(found[0])
    assert found[2][-4:] == ["2", "2", "1", "0"]
    assert found[3][-3:] == ["1", "16", "0"]  # added residual


def test_a_sum_that_nobody_reads_is_not_written():
    x = _t("x", 8, 64)
    total, y = ops.residual_norm("rms")(x, _t("r", 8, 64))
    line = next(l for l in _plan(y) if l.startswith("op residual_norm"))
    assert " 4 0 2 0 0 2 " in line
    total, y = ops.residual_norm("rms")(x, _t("r2", 8, 64))
    assert " 4 0 2 0 1 2 " in next(l for l in _plan(total, y) if l.startswith("op residual_norm"))


X8, W8 = lambda: _t("x", 4, 32, dtype="int8"), lambda: _t("w", 16, 32, dtype="int8")  # noqa: E731
S4, S16 = lambda: _t("xs", 4, dtype="float32"), lambda: _t("ws", 16, dtype="float32")  # noqa: E731


@pytest.mark.parametrize("build,said", [
    (lambda: ops.gemm_rcr_i8("square"), "unknown epilogue"), (lambda: ops.gemm_rcr_i8(dtype="float32"), "float16 or bfloat16"),
    (lambda: ops.gemm_rcr_i8()(X8(), W8(), S16()), "needs x_scale"), (lambda: ops.gemm_rcr_i8()(_t("x", 4, 32), W8(), S16(), S4()), "goes with an int8"),
    (lambda: ops.gemm_rcr_i8()(_t("x", 4, 31, dtype="int8"), W8(), S16(), S4()), "static N and K"),
    (lambda: ops.gemm_rcr_i8()(X8(), _t("w", 16, 32), S16(), S4()), "w must be int8"), (lambda: ops.gemm_rcr_i8()(X8(), W8(), S4(), S4()), "w_scale"),
    (lambda: ops.gemm_rcr_i8()(X8(), W8(), S16(), _t("s", 4)), "x_scale"), (lambda: ops.gemm_rcr_i8("add")(X8(), W8(), S16(), S4()), "needs d0"),
    (lambda: ops.gemm_rcr_i8()(X8(), W8(), S16(), S4(), d0=_t("d", 4, 16)), "takes no d0"),
    (lambda: ops.gemm_rcr_i8(dtype="bfloat16")(X8(), W8(), S16(), S4(), bias=_t("b", 16)), "bias must be"),
    (lambda: ops.gemm_rcr_i8()(_t("x", 2, 131072, dtype="int8"), _t("w", 2, 131072, dtype="int8"), _t("s", 2, dtype="float32"), S4()), "131071"),
    (lambda: ops.quantize_rows("elu"), "unknown activation"), (lambda: ops.quantize_rows()(X8()), "float16 or bfloat16"),
    (lambda: ops.quantize_rows(gated=True)(_t("x", 4, 33)), "two halves"), (lambda: ops.quantize_rows()(_t("x", 32)), "static columns"),
    (lambda: ops.quantize_rows()(_t("x", 4, IntVar([1, 9], name="k"))), "static columns"),
    (lambda: ops.residual_norm("batch"), "a norm is"), (lambda: ops.residual_norm(post_norm="batch"), "a norm is"),
    (lambda: ops.residual_norm()(_t("x", 4, 32), _t("r", 4, 31)), "does not fit"), (lambda: ops.residual_norm()(_t("x", 4, 32), gate=_t("g", 31)), "does not fit"),
    (lambda: ops.residual_norm()(_t("x", 4, 32), gamma=_t("g", 32, dtype="bfloat16")), "does not fit"),
    (lambda: ops.residual_norm()(_t("x", 4, 32), post_gamma=_t("g", 32)), "need a post_norm"),
    (lambda: ops.residual_norm(post_norm="rms")(_t("x", 4, 32), post_gamma=_t("g", 2, 32)), "does not fit"),
    (lambda: ops.residual_norm()(X8()), "float16 or bfloat16"),
])
def test_refusals(build, said):
    with pytest.raises(RuntimeError, match=said):
        build()
