"""What 8-bit serving of a transformer block costs: the int8 product with a scale per token and per channel, the quantisation of
rows in front of it (plain, or of a gated feed-forward's two halves), and the norms around a block with its gate and residual.

listed() names a fixed set, draw() gives more of the same ranges; prepare() makes what a program holds before the call, run() is one
pass, work() what it cannot do without, exact() the same outputs in 64 bits from the operators' definitions.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_ACTIVATIONS = ("identity", "relu", "gelu", "swish")
# epilogues of the product: (activation of acc * scales + bias, how the residual joins)
_EPILOGUES = {"": ("identity", None), "relu": ("relu", None), "gelu": ("gelu", None), "swish": ("swish", None),
              "add": ("identity", "add"), "mul": ("identity", "mul")}


def listed():
    return [
        # one token through a square projection: what a decoder waits for, token by token
        {"name": "product_1_row", "op": "product", "rows": 1, "columns": 4096, "depth": 4096, "epilogue": "", "bias": False, "dtype": "fp16"},
        # a batch of requests, a token each, against a large matrix, onto the residual stream
        {"name": "product_24_rows", "op": "product", "rows": 24, "columns": 8192, "depth": 8192, "epilogue": "add", "bias": True, "dtype": "bf16"},
        # sizes that no tile divides, rows of the operands padded to 16 bytes
        {"name": "product_odd", "op": "product", "rows": 777, "columns": 1283, "depth": 2041, "epilogue": "relu", "bias": True, "dtype": "fp16"},
        # a long prompt through the largest matrix
        {"name": "product_large", "op": "product", "rows": 16384, "columns": 8192, "depth": 8192, "epilogue": "gelu", "bias": True, "dtype": "bf16"},
        # eight tokens of activations in 16 bits, quantised on the way into the product
        {"name": "linear_8_rows", "op": "linear", "rows": 8, "columns": 4096, "depth": 4096, "activation": "identity", "gated": False, "dtype": "bf16"},
        # the second half of a gated feed-forward over a prompt: activation, product of the halves, quantisation, projection
        {"name": "linear_gated", "op": "linear", "rows": 4096, "columns": 4096, "depth": 8192, "activation": "swish", "gated": True, "dtype": "bf16"},
        # the same for a ragged batch and an odd width
        {"name": "linear_gated_odd", "op": "linear", "rows": 333, "columns": 1000, "depth": 2733, "activation": "gelu", "gated": True, "dtype": "fp16"},
        # a few decoding sequences, norm before the next block
        {"name": "norm_16_rows", "op": "norm", "rows": 16, "columns": 4096, "norm": "rms", "post": "", "gate": 0, "affine": False, "dtype": "bf16"},
        # an encoder's batch of 64 sequences of 384 tokens
        {"name": "norm_encoder", "op": "norm", "rows": 24576, "columns": 768, "norm": "layer", "post": "", "gate": 0, "affine": True, "dtype": "fp16"},
        # an image block with a gate per sample and norms on both sides
        {"name": "norm_gated", "op": "norm", "rows": 8192, "columns": 1280, "norm": "layer", "post": "rms", "gate": 8, "affine": True, "dtype": "bf16"},
        # the norm of a decoding step straight into an 8-bit projection
        {"name": "norm_linear_4_rows", "op": "norm_linear", "rows": 4, "columns": 2048, "width": 2048, "norm": "rms", "post": "", "gate": 0, "affine": False, "dtype": "fp16"},
        # the same for a prompt, with both norms and a gate per channel
        {"name": "norm_linear_prompt", "op": "norm_linear", "rows": 8192, "columns": 4096, "width": 1024, "norm": "rms", "post": "rms", "gate": 1, "affine": False, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Sizes as models have them (multiples of 64) three times out of four, any other size else."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(("product", "product", "linear", "norm", "norm_linear"))
    dtype = rng.choice(sorted(_TYPES))
    if op == "product":
        rows, columns, depth = _spread(rng, 1, 16384), _width(rng, 64, 8192), _width(rng, 64, 8192)
        return {"op": op, "rows": rows, "columns": columns, "depth": depth, "epilogue": rng.choice(sorted(_EPILOGUES)),
                "bias": rng.random() < 0.5, "dtype": dtype}
    if op == "linear":
        rows, columns, depth = _spread(rng, 1, 8192), _width(rng, 64, 8192), _width(rng, 64, 8192)
        return {"op": op, "rows": rows, "columns": columns, "depth": depth, "activation": rng.choice(_ACTIVATIONS),
                "gated": rng.random() < 0.5, "dtype": dtype}
    gate = rng.choice((0, 1, 4))
    rows = _spread(rng, 1, 16384)
    rows = rows if gate < 2 else max(gate, rows // gate * gate)
    case = {"op": op, "rows": rows, "columns": _width(rng, 64, 8192), "norm": rng.choice(("layer", "rms")),
            "post": rng.choice(("", "layer", "rms")), "gate": gate, "affine": rng.random() < 0.5, "dtype": dtype}
    if op == "norm_linear":
        case["width"] = _width(rng, 64, 2048)
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _int8(g, rows, depth):
    """Rows of 8-bit values as quantised normal values lie, at a pitch of whole 16 bytes, the way a program stores them."""
    store = torch.zeros(rows, (depth + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    store[:, :depth] = (torch.randn(rows, depth, generator=g, device="cuda") * 32).round_().clamp_(-127, 127)
    return store[:, :depth]


def _weights(g, columns, depth):
    scale = (torch.rand(columns, generator=g, device="cuda") + 0.5) / (32 * math.sqrt(depth))
    return {"w": _int8(g, columns, depth), "w_scale": scale}


def prepare(case, seed):
    g, dtype = _generator(seed), _TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "product":
        rows, columns, depth = case["rows"], case["columns"], case["depth"]
        s |= _weights(g, columns, depth)
        s["x"] = _int8(g, rows, depth)
        s["x_scale"] = (torch.rand(rows, generator=g, device="cuda") + 0.5) / 32
        s["bias"] = _normal(g, columns, scale=0.5, dtype=dtype) if case["bias"] else None
        s["d0"] = _normal(g, rows, columns, dtype=dtype) if _EPILOGUES[case["epilogue"]][1] else None
        return s
    if case["op"] == "linear":
        s |= _weights(g, case["columns"], case["depth"])
        s["x"] = _normal(g, case["rows"], case["depth"] * (2 if case["gated"] else 1), dtype=dtype)
        return s
    rows, columns, gate = case["rows"], case["columns"], case["gate"]
    s["x"] = _normal(g, rows, columns, scale=2.0, shift=0.25, dtype=dtype)
    s["residual"] = _normal(g, rows, columns, scale=3.0, dtype=dtype)
    s["gate"] = _normal(g, *((gate, columns) if gate > 1 else (columns,)), scale=0.5, shift=0.5, dtype=dtype) if gate else None
    s["post_gamma"] = _normal(g, columns, scale=0.1, shift=1.0, dtype=dtype) if case["post"] else None
    s["gamma"] = _normal(g, columns, scale=0.1, shift=1.0, dtype=dtype)
    s["beta"] = _normal(g, columns, scale=0.1, dtype=dtype) if case["affine"] else None
    if case["op"] == "norm_linear":
        s |= _weights(g, case["width"], columns)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _activate(name, v):
    if name == "relu":
        return v.clamp(min=0)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "swish":
        return v / (1 + torch.exp(-v))
    return v


def _product(x, x_scale, s, bias=None, d0=None, epilogue=""):
    """x [rows, depth] of whole numbers in 32 bits, x_scale [rows, 1]; the result in 32 bits."""
    y = (x @ s["w"].float().T) * x_scale * s["w_scale"]
    if bias is not None:
        y = y + bias.float()
    activation, joins = _EPILOGUES[epilogue]
    y = _activate(activation, y)
    return y + d0.float() if joins == "add" else y * d0.float() if joins == "mul" else y


def _quantised(v):
    """(whole numbers, scale) of the rows of v, all in 32 bits."""
    most = v.abs().amax(-1, keepdim=True)
    q = torch.where(most > 0, torch.round(127 * v / most), torch.zeros_like(v))
    return q, most / 127


def _normed(kind, v, gamma, beta=None, eps=1e-5):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * gamma.float()
    return v if beta is None else v + beta.float()


def _summed(s):
    case, p = s["case"], s["x"].float()
    if case["post"]:
        p = _normed(case["post"], p, s["post_gamma"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        p = p * (gate if gate.dim() == 1 else gate.repeat_interleave(case["rows"] // gate.shape[0], 0))
    return 0.75 * s["residual"].float() + p


def _plain(s):
    case = s["case"]
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "product":
        return _product(s["x"].float(), s["x_scale"][:, None], s, s["bias"], s["d0"], case["epilogue"]).to(dtype)
    if case["op"] == "linear":
        v = s["x"].float()
        if case["gated"]:
            v = _activate(case["activation"], v[:, :case["depth"]]) * v[:, case["depth"]:]
        else:
            v = _activate(case["activation"], v)
        return _product(*_quantised(v), s).to(dtype)
    total = _summed(s)
    y = _normed(case["norm"], total, s["gamma"], s["beta"])
    if case["op"] == "norm":
        return total.to(dtype), y.to(dtype)
    return total.to(dtype), _product(*_quantised(y), s).to(dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _calls(s):
    from aitemplate_b200 import kernels

    case = s["case"]
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "product":
        return kernels.gemm_rcr_i8(s["x"], s["w"], s["w_scale"], s["x_scale"], bias=s["bias"], d0=s["d0"], epilogue=case["epilogue"], dtype=dtype)
    if case["op"] == "linear":
        if case["gated"] or case["activation"] != "identity":
            q, scale = kernels.quantize_rows(s["x"], case["activation"], gated=case["gated"])
            return kernels.gemm_rcr_i8(q, s["w"], s["w_scale"], scale, dtype=dtype)
        return kernels.gemm_rcr_i8(s["x"], s["w"], s["w_scale"])
    arguments = dict(residual=s["residual"], gate=s["gate"], post_gamma=s["post_gamma"], gamma=s["gamma"], beta=s["beta"],
                     post_norm=case["post"] or None, norm=case["norm"], residual_scale=0.75)
    if case["op"] == "norm":
        return kernels.residual_norm(s["x"], **arguments)
    total, q, scale = kernels.residual_norm(s["x"], quantize=True, **arguments)
    return total, kernels.gemm_rcr_i8(q, s["w"], s["w_scale"], scale, dtype=dtype)


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    rows = case["rows"]
    if case["op"] == "product":
        columns, depth = case["columns"], case["depth"]
        moved = rows * depth + columns * depth + 4 * rows + 4 * columns + 2 * rows * columns
        moved += (2 * columns if case["bias"] else 0) + (2 * rows * columns if _EPILOGUES[case["epilogue"]][1] else 0)
        return {"bytes": moved, "flops": 2 * rows * columns * depth}
    if case["op"] == "linear":
        columns, depth = case["columns"], case["depth"]
        moved = 2 * rows * depth * (2 if case["gated"] else 1) + columns * depth + 4 * columns + 2 * rows * columns
        return {"bytes": moved, "flops": 2 * rows * columns * depth}
    columns = case["columns"]
    moved = 6 * rows * columns + 2 * columns * (1 + (1 if case["post"] else 0) + (1 if case["affine"] else 0) + case["gate"])
    if case["op"] == "norm":
        return {"bytes": moved + 2 * rows * columns, "flops": 16 * rows * columns}
    width = case["width"]
    return {"bytes": moved + width * columns + 4 * width + 2 * rows * width, "flops": 2 * rows * columns * width}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}

    def act(name, v):
        return {"identity": lambda: v, "relu": lambda: torch.where(v > 0, v, 0 * v), "gelu": lambda: v * torch.special.ndtr(v),
                "swish": lambda: v * torch.sigmoid(v)}[name]()

    def to_8_bits(v):
        most = torch.linalg.vector_norm(v, ord=math.inf, dim=1)
        steps = torch.div(v * 127, torch.where(most == 0, torch.ones_like(most), most)[:, None])
        return torch.round(steps), most / 127

    def times_weights(q, scale):
        return torch.einsum("mk,nk->mn", q, d["w"]) * torch.outer(scale, d["w_scale"])

    def norm(kind, v, gamma, beta):
        centre = v.sum(1) / v.shape[1] if kind == "layer" else torch.zeros_like(v[:, 0])
        away = v - centre[:, None]
        spread = torch.sqrt(torch.einsum("mn,mn->m", away, away) / v.shape[1] + 1e-5)
        return away / spread[:, None] * gamma + (beta if beta is not None else 0)

    if case["op"] == "product":
        y = times_weights(d["x"], d["x_scale"]) + d.get("bias", 0)
        activation, joins = _EPILOGUES[case["epilogue"]]
        y = act(activation, y)
        return y if joins is None else torch.add(y, d["d0"]) if joins == "add" else torch.mul(y, d["d0"])
    if case["op"] == "linear":
        halves = d["x"].split(case["depth"], 1)
        v = act(case["activation"], halves[0])
        return times_weights(*to_8_bits(v * halves[1] if case["gated"] else v))
    p = norm(case["post"], d["x"], d["post_gamma"], None) if case["post"] else d["x"]
    if case["gate"]:
        parts = d["gate"].reshape(max(1, case["gate"]), 1, -1)
        p = (p.reshape(parts.shape[0], -1, case["columns"]) * parts).reshape(p.shape)
    total = d["residual"] * 0.75 + p
    y = norm(case["norm"], total, d["gamma"], d.get("beta"))
    return (total, y) if case["op"] == "norm" else (total, times_weights(*to_8_bits(y)))
