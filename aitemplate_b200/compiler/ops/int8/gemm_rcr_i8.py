"""gemm_rcr_i8 graph node: a gemm_rcr of signed 8-bit integers with a scale per row of either operand.

    y = gemm_rcr_i8(epilogue="", dtype=None)(x, w, w_scale, x_scale, bias, d0, d1)
      = epilogue((x w^T) * x_scale[:, None] * w_scale + bias, d0, d1)

w is int8 [N, K] with w_scale float32 [N]. x is int8 [..., K] with x_scale float32 [...] (quantize_rows, residual_norm), or has 16 bits
and no x_scale: then its rows are quantised on the way. `epilogue` is the suffix of the gemm_rcr_bias_<suffix> ops ("" for none); bias
is optional, d0 and d1 are what the epilogue takes. `dtype`: of y, bias, d0 and d1 (default: x's if that has 16 bits, else d0's or the
bias's, else float16). Sums are exact, so the result does not depend on how it is computed; the tensor cores take rows of a multiple
of 16 elements, others go to a slower kernel (pad x and w with zeros). The reference's GEMMs take 16- and 32-bit floats only."""
from __future__ import annotations

from typing import Any, Dict, Optional

from ...base import IntImm, Operator, Tensor
from .quantize_rows import ACTIVATIONS

_BINARY = {None: 0, "add": 1, "mul": 2}
# suffix -> (activation, joins d0, joins d1, activation behind)
EPILOGUES = {a if a != "identity" else "": (a, None, None, "identity") for a in ACTIVATIONS}
EPILOGUES.update({
    "add": ("identity", "add", None, "identity"), "add_relu": ("identity", "add", None, "relu"),
    "add_add": ("identity", "add", "add", "identity"), "add_add_relu": ("identity", "add", "add", "relu"),
    "mul": ("identity", "mul", None, "identity"), "mul_add": ("identity", "mul", "add", "identity"),
    "mul_tanh": ("identity", "mul", None, "tanh"), "sigmoid_mul": ("sigmoid", "mul", None, "identity"),
    "sigmoid_mul_tanh": ("sigmoid", "mul", None, "tanh"),
})


class gemm_rcr_i8(Operator):
    def __init__(self, epilogue: str = "", dtype: Optional[str] = None) -> None:
        super().__init__()
        if epilogue not in EPILOGUES:
            raise RuntimeError(f"gemm_rcr_i8: unknown epilogue {epilogue}")
        if dtype not in (None, "float16", "bfloat16"):
            raise RuntimeError(f"gemm_rcr_i8: the result is float16 or bfloat16, got {dtype}")
        self._attrs["op"] = "gemm_rcr_i8"
        self._attrs["has_profiler"] = False
        self._attrs["epilogue"] = epilogue
        self._attrs["dtype"] = dtype

    def _get_op_attributes(self):
        return {"epilogue": self._attrs["epilogue"], "dtype": self._attrs["dtype"]}

    def __call__(self, x: Tensor, w: Tensor, w_scale: Tensor, x_scale: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                 d0: Optional[Tensor] = None, d1: Optional[Tensor] = None) -> Tensor:
        xs, ws = x._attrs["shape"], w._attrs["shape"]
        if len(xs) < 2 or len(ws) != 2 or not all(isinstance(d, IntImm) for d in (xs[-1], *ws)) or xs[-1] != ws[1]:
            raise RuntimeError(f"gemm_rcr_i8: x [..., K] and w [N, K] with static N and K, got {xs} and {ws}")
        if not 0 < ws[1].value() < 1 << 17:
            raise RuntimeError(f"gemm_rcr_i8: K is 1 to 131071, got {ws[1].value()}")
        if w.dtype() != "int8":
            raise RuntimeError(f"gemm_rcr_i8: w must be int8, got {w.dtype()}")
        if x.dtype() == "int8":
            if x_scale is None:
                raise RuntimeError("gemm_rcr_i8: an int8 x needs x_scale")
        elif x.dtype() not in ("float16", "bfloat16"):
            raise RuntimeError(f"gemm_rcr_i8: x must be int8, float16 or bfloat16, got {x.dtype()}")
        elif x_scale is not None:
            raise RuntimeError(f"gemm_rcr_i8: x_scale goes with an int8 x, got {x.dtype()}")
        for name, t, shape in (("w_scale", w_scale, [ws[0]]), ("x_scale", x_scale, list(xs[:-1]))):
            if t is not None and (t.dtype() != "float32" or list(t._attrs["shape"]) != shape):
                raise RuntimeError(f"gemm_rcr_i8: {name} must be float32 of shape {shape}, got {t.dtype()} {t._attrs['shape']}")
        given = [t.dtype() for t in (x, d0, bias) if t is not None and t.dtype() != "int8"]
        dtype = self._attrs["dtype"] or (given[0] if given else "float16")
        _, b1, b2, _ = EPILOGUES[self._attrs["epilogue"]]
        out_shape = list(xs[:-1]) + [ws[0]]
        for name, t, wanted, shape in (("bias", bias, bias is not None, [ws[0]]), ("d0", d0, b1 is not None, out_shape),
                                       ("d1", d1, b2 is not None, out_shape)):
            if wanted != (t is not None):
                raise RuntimeError(f"gemm_rcr_i8: the epilogue '{self._attrs['epilogue']}' {'needs' if wanted else 'takes no'} {name}")
            if t is not None and (t.dtype() != dtype or list(t._attrs["shape"]) != shape):
                raise RuntimeError(f"gemm_rcr_i8: {name} must be {dtype} of shape {shape}, got {t.dtype()} {t._attrs['shape']}")
        self._operands = [x, x_scale, w, w_scale, bias, d0, d1]
        self._attrs["inputs"] = [t for t in self._operands if t is not None]
        self._set_depth()
        y = Tensor(out_shape, src_ops={self}, dtype=dtype)
        self._attrs["outputs"] = [y]
        return y

    def _lower(self) -> Dict[str, Any]:
        # (a pass may have put another tensor in an input's place: the operands are what is there now)
        now = iter(self._attrs["inputs"])
        operands = [None if t is None else next(now) for t in self._operands]
        u1, b1, b2, u2 = EPILOGUES[self._attrs["epilogue"]]
        code = ACTIVATIONS[u1] | (_BINARY[b1] << 4) | (_BINARY[b2] << 6) | (ACTIVATIONS[u2] << 8)
        return {"kernel": "gemm_rcr_i8", "operands": operands, "ints": [code], "floats": []}
