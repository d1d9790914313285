"""quantize_rows graph node: rows of 16-bit activations to signed 8-bit integers with an fp32 scale each.

    q, scale = quantize_rows(activation="identity", gated=False)(x)

scale = max |v| / 127 and q = round(127 v / max |v|), ties to even, with v = act(x), or with `gated` v = act(x[..., :n]) * x[..., n:]
for the two halves of a gated feed-forward's first product. q and scale are operands of gemm_rcr_i8. A row of v that is all zeros has
scale 0, one with an infinity or a NaN in it scale NaN (and q 0). The reference has no 8-bit activations; the activations are those of
its GEMM epilogues."""
from __future__ import annotations

from typing import Any, Dict, Tuple

from ...base import IntImm, Operator, Tensor

ACTIVATIONS = {"identity": 0, "relu": 1, "gelu": 2, "fast_gelu": 3, "sigmoid": 4, "tanh": 5, "swish": 6, "hardswish": 7}


class quantize_rows(Operator):
    def __init__(self, activation: str = "identity", gated: bool = False) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise RuntimeError(f"quantize_rows: unknown activation {activation}")
        self._attrs["op"] = "quantize_rows"
        self._attrs["has_profiler"] = False
        self._attrs["activation"] = activation
        self._attrs["gated"] = bool(gated)

    def _get_op_attributes(self):
        return {"activation": self._attrs["activation"], "gated": self._attrs["gated"]}

    def __call__(self, x: Tensor) -> Tuple[Tensor, Tensor]:
        shape = x._attrs["shape"]
        if len(shape) < 2 or not isinstance(shape[-1], IntImm):
            raise RuntimeError(f"quantize_rows: x must be [..., columns] with static columns, got {shape}")
        if x.dtype() not in ("float16", "bfloat16"):
            raise RuntimeError(f"quantize_rows: x must be float16 or bfloat16, got {x.dtype()}")
        n = shape[-1].value()
        if self._attrs["gated"]:
            if n % 2:
                raise RuntimeError(f"quantize_rows: the rows of a gated x have two halves, got {n} columns")
            n //= 2
        if n == 0:
            raise RuntimeError("quantize_rows: x has no columns")
        self._attrs["inputs"] = [x]
        self._set_depth()
        q = Tensor(list(shape[:-1]) + [IntImm(n)], src_ops={self}, dtype="int8")
        scale = Tensor(list(shape[:-1]), src_ops={self}, dtype="float32")
        self._attrs["outputs"] = [q, scale]
        return q, scale

    def _lower(self) -> Dict[str, Any]:
        return {"kernel": "quantize_rows", "operands": list(self._attrs["inputs"]),
                "ints": [ACTIVATIONS[self._attrs["activation"]], int(self._attrs["gated"])], "floats": []}
