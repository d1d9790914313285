"""residual_norm graph node: what stands between two blocks of a transformer, in one pass over the rows.

    total, y = residual_norm(norm="layer", post_norm=None, residual_scale=1.0, eps=1e-5)(
        x, residual, gate, post_gamma, post_beta, gamma, beta)

      p = post_norm(x) * post_gamma + post_beta;  total = residual_scale * residual + gate * p;  y = norm(total) * gamma + beta

norm and post_norm are "layer" or "rms" over the last dim, post_norm None for no norm after the block; every operand but x may be None.
post_gamma and post_beta are [N]; gate, gamma and beta [N] or [G, N], a vector for each of G equal parts of the rows (a gate per
sample). With quantize=True the outputs are (total, q, scale): y as int8 rows with a float32 scale each, operands of gemm_rcr_i8.
Next of kin in the reference: layernorm (python/aitemplate/compiler/ops/layernorm/layernorm.py:58-450) behind an elementwise add."""
from __future__ import annotations

from typing import Any, Dict, Optional

from ...base import IntImm, Operator, Tensor

NORMS = {None: 0, "layer": 1, "rms": 2}


class residual_norm(Operator):
    def __init__(self, norm: str = "layer", post_norm: Optional[str] = None, residual_scale: float = 1.0, eps: float = 1e-5,
                 quantize: bool = False) -> None:
        super().__init__()
        if norm not in ("layer", "rms") or post_norm not in NORMS:
            raise RuntimeError(f"residual_norm: a norm is 'layer' or 'rms', got {norm!r} and {post_norm!r}")
        self._attrs["op"] = "residual_norm"
        self._attrs["has_profiler"] = False
        self._attrs.update(norm=norm, post_norm=post_norm, residual_scale=float(residual_scale), eps=float(eps), quantize=bool(quantize))

    def _get_op_attributes(self):
        return {k: self._attrs[k] for k in ("norm", "post_norm", "residual_scale", "eps", "quantize")}

    def __call__(self, x: Tensor, residual: Optional[Tensor] = None, gate: Optional[Tensor] = None,
                 post_gamma: Optional[Tensor] = None, post_beta: Optional[Tensor] = None, gamma: Optional[Tensor] = None,
                 beta: Optional[Tensor] = None):
        shape = x._attrs["shape"]
        if len(shape) < 2 or not isinstance(shape[-1], IntImm) or shape[-1].value() == 0:
            raise RuntimeError(f"residual_norm: x must be [..., N] with a static N, got {shape}")
        if x.dtype() not in ("float16", "bfloat16"):
            raise RuntimeError(f"residual_norm: x must be float16 or bfloat16, got {x.dtype()}")
        if self._attrs["post_norm"] is None and (post_gamma is not None or post_beta is not None):
            raise RuntimeError("residual_norm: post_gamma and post_beta need a post_norm")
        self._operands = [x, residual, gate, post_gamma, post_beta, gamma, beta]
        for name, t in zip(("residual", "gate", "post_gamma", "post_beta", "gamma", "beta"), self._operands[1:]):
            if t is None:
                continue
            s = t._attrs["shape"]
            if name == "residual":
                fits = list(s) == list(shape)
            else:
                fits = len(s) in ((1,) if name.startswith("post") else (1, 2)) and all(isinstance(d, IntImm) for d in s) and s[-1] == shape[-1]
            if not fits or t.dtype() != x.dtype():
                raise RuntimeError(f"residual_norm: {name} ({t.dtype()} {s}) does not fit x ({x.dtype()} {shape})")
        self._attrs["inputs"] = [t for t in self._operands if t is not None]
        self._set_depth()
        total = Tensor(list(shape), src_ops={self}, dtype=x.dtype())
        outputs = [total, Tensor(list(shape), src_ops={self}, dtype="int8" if self._attrs["quantize"] else x.dtype())]
        if self._attrs["quantize"]:
            outputs.append(Tensor(list(shape[:-1]), src_ops={self}, dtype="float32"))
        self._attrs["outputs"] = outputs
        return tuple(outputs)

    def _lower(self) -> Dict[str, Any]:
        now = iter(self._attrs["inputs"])
        operands = [None if t is None else next(now) for t in self._operands]
        total = self._attrs["outputs"][0]
        used = bool(total._attrs["dst_ops"]) or total._attrs["is_output"]  # nobody reads it: it is not written
        return {"kernel": "residual_norm", "operands": operands,
                "ints": [NORMS[self._attrs["post_norm"]], NORMS[self._attrs["norm"]], int(self._attrs["quantize"]), int(used)],
                "floats": [self._attrs["residual_scale"], self._attrs["eps"]]}
