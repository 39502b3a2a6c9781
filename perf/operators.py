"""The 8-bit feed-forward operators as a serving program calls them, one call at a time, for measuring them.

Four operators, which together are one feed-forward layer on 8-bit weights: the norm that joins the residual and leaves
8-bit rows (`norm`), the gate and up products with SwiGLU and 8-bit rows as output (`gate_up`), the product on 8-bit
operands (`linear`), and the quantisation of rows that no norm made, or of a checkpoint's matrix (`quantize`).

8-bit rows are e4m3 values with a float32 scale for each row and 128 columns; an 8-bit weight has a scale for each 128
features and 128 columns.  The last block of a row may be short.  Rows of 8-bit values lie at multiples of 16 bytes.

Sizes are those of this repository's three benchmark models (hidden 1,024 / 1,280 / 3,072, intermediate 2,048 / 3,072 /
12,288), its batch sizes and prompt lengths, and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False             # whether `run` calls the framework's kernels

BLOCK = 128
LARGEST = 448.0         # of e4m3
TINY = 2.0 ** -126      # the smallest scale
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _norm(name, rows, width, dtype, other, residual):
    case = {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "other": other, "residual": residual}
    return {"name": name, **case} if name else case


def _quantize(name, rows, width, dtype, block_rows):
    case = {"op": "quantize", "rows": rows, "width": width, "dtype": dtype, "block_rows": block_rows}
    return {"name": name, **case} if name else case


def _linear(name, rows, features, width, dtype, bias):
    case = {"op": "linear", "rows": rows, "features": features, "width": width, "dtype": dtype, "bias": bias}
    return {"name": name, **case} if name else case


def _gate_up(name, rows, features, width):
    case = {"op": "gate_up", "rows": rows, "features": features, "width": width}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user's chat: the norm in front of the smallest model's feed-forward, both mixers' outputs joining the residual
        _norm("norm-1", 1, 1024, "bfloat16", True, True),
        # a full prompt step of the largest model
        _norm("norm-8192-large", 8192, 3072, "bfloat16", True, True),
        # a float32 engine, a width that is no multiple of a block or of a vector, nothing to join but the residual
        _norm("norm-777-odd", 777, 1003, "float32", False, True),
        # a prompt's mixer outputs on the way to an 8-bit output projection
        _quantize("quantize-rows-2048", 2048, 1536, "bfloat16", 1),
        # a checkpoint's matrix as it is laid out at load
        _quantize("quantize-weight-large", 12288, 3072, "bfloat16", 128),
        # the smallest product: one token through the smallest model's down projection
        _linear("down-1", 1, 1024, 2048, "bfloat16", False),
        # a full server's decode step, the largest model's down projection: bound by reading the weight
        _linear("down-64-large", 64, 3072, 12288, "bfloat16", False),
        # a short prompt, sizes that are multiples of nothing, a bias, float32 out
        _linear("linear-203-odd", 203, 1003, 1431, "float32", True),
        # a full prompt step, the largest model's down projection: bound by the tensor cores
        _linear("down-8192-large", 8192, 3072, 12288, "bfloat16", False),
        # a small server's decode step at the middle model
        _gate_up("gate-up-8", 8, 3072, 1280),
        # a full server's decode step of the largest model
        _gate_up("gate-up-64-large", 64, 12288, 3072),
        # a full prompt step of the largest model: the most work
        _gate_up("gate-up-8192-large", 8192, 12288, 3072),
    ]


def _between(rng, low, high):
    """A size from low to high, spread over its logarithm; a third of them rounded to a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.33 and n >= 64:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "gate_up", "gate_up"])
    rows, dtype = _between(rng, 1, 8192), rng.choice(["bfloat16", "float32"])
    if op == "norm":
        return _norm(None, rows, _between(rng, 64, 3072), dtype, rng.random() < 0.5, rng.random() < 0.8)
    if op == "quantize":
        if rng.random() < 0.5:
            return _quantize(None, rows, _between(rng, 64, 12288), dtype, 1)
        return _quantize(None, _between(rng, 64, 12288), _between(rng, 64, 3072), dtype, 128)
    if op == "linear":
        return _linear(None, rows, _between(rng, 64, 3072), _between(rng, 64, 12288), dtype, rng.random() < 0.3)
    return _gate_up(None, rows, _between(rng, 64, 12288), _between(rng, 64, 3072))


# ------------------------------------------------------------------ plain forms
def _blocks(v, block_rows):
    """[rows, width] as [row blocks, block_rows, column blocks, 128], filled up with zeros."""
    rows, width = v.shape
    more_rows, more = -rows % block_rows, -width % BLOCK
    v = torch.nn.functional.pad(v, (0, more, 0, more_rows))
    return v.view(v.shape[0] // block_rows, block_rows, v.shape[1] // BLOCK, BLOCK)


def _to_8_bits(v, block_rows=1):
    """(e4m3 values, float32 scales per block) of a float32 matrix."""
    rows, width = v.shape
    b = _blocks(v, block_rows)
    scales = (b.abs().amax((1, 3)) / LARGEST).clamp(min=TINY)
    q = (b / scales[:, None, :, None]).reshape(b.shape[0] * block_rows, -1)[:rows, :width]
    return q.to(torch.float8_e4m3fn), scales


def _spread(scales, block_rows, rows, width):
    """The scale of every element."""
    if block_rows > 1:
        scales = scales.repeat_interleave(block_rows, 0)[:rows]
    return scales.repeat_interleave(BLOCK, 1)[:, :width]


def _from_8_bits(q, scales, block_rows=1):
    return q.float() * _spread(scales, block_rows, *q.shape)


# ------------------------------------------------------------------ inputs
def _aligned(q):
    """The same 8-bit values with rows at multiples of 16 bytes."""
    rows, width = q.shape
    out = torch.zeros((rows, -(-width // 16) * 16), dtype=torch.uint8, device=q.device).view(torch.float8_e4m3fn)
    out[:, :width].view(torch.uint8).copy_(q.view(torch.uint8))
    return out[:, :width]


def _activations(rows, width, gen):
    """Rows as a norm or a gated product leaves them: a few columns much larger than the others."""
    x = torch.randn((rows, width), generator=gen, device="cuda")
    loud = torch.rand((width,), generator=gen, device="cuda") < 0.01
    return x * torch.where(loud, 8.0, 1.0)


def _weight(features, width, gen):
    """A checkpoint's matrix: features of differing size."""
    w = torch.randn((features, width), generator=gen, device="cuda") * width ** -0.5
    return w * torch.exp(0.3 * torch.randn((features, 1), generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    op, rows, width = case["op"], case["rows"], case["width"]
    state = {"op": op}
    if op == "norm":
        dtype = _DTYPES[case["dtype"]]
        state["x"] = _activations(rows, width, gen).to(dtype)
        for name in ("other", "residual"):
            state[name] = _activations(rows, width, gen).to(dtype) if case[name] else None
        state["weight"] = 1.0 + 0.1 * torch.randn((width,), generator=gen, device="cuda")
        state["in_scales"] = (0.8, 0.7) if case["other"] else (1.0, 1.0)
        state["eps"], state["out_scale"] = 1e-5, 1.0
    elif op == "quantize":
        made = _activations if case["block_rows"] == 1 else _weight
        state["x"], state["block_rows"] = made(rows, width, gen).to(_DTYPES[case["dtype"]]), case["block_rows"]
    else:
        q, scales = _to_8_bits(_activations(rows, width, gen))
        # the scales of one column block lie together, as the operators that make 8-bit rows leave them
        state["x"], state["x_scales"] = _aligned(q), scales.t().contiguous().t()
        for name in ("w",) if op == "linear" else ("gate", "up"):
            q, scales = _to_8_bits(_weight(case["features"], width, gen), BLOCK)
            state[name], state[name + "_scales"] = _aligned(q), scales
        if op == "linear":
            state["bias"] = torch.randn((case["features"],), generator=gen, device="cuda") if case["bias"] else None
            state["out_scale"], state["dtype"] = 1.1, _DTYPES[case["dtype"]]
        else:
            state["act_scale"] = 0.9
    return state


# ------------------------------------------------------------------ one pass
def _plain(s):
    op = s["op"]
    if op == "norm":
        r = s["x"].float() * s["in_scales"][0]
        if s["other"] is not None:
            r = r + s["other"].float() * s["in_scales"][1]
        if s["residual"] is not None:
            r = r + s["residual"].float()
        n = r * torch.rsqrt((r * r).mean(1, keepdim=True) + s["eps"]) * s["weight"] * s["out_scale"]
        q, scales = _to_8_bits(n)
        return {"values": q, "scales": scales, "residual": r.to(s["x"].dtype)}
    if op == "quantize":
        q, scales = _to_8_bits(s["x"].float(), s["block_rows"])
        return {"values": q, "scales": scales}
    x = _from_8_bits(s["x"], s["x_scales"])
    if op == "linear":
        y = x @ _from_8_bits(s["w"], s["w_scales"], BLOCK).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return {"y": (y * s["out_scale"]).to(s["dtype"])}
    gate = x @ _from_8_bits(s["gate"], s["gate_scales"], BLOCK).t() * s["act_scale"]
    up = x @ _from_8_bits(s["up"], s["up_scales"], BLOCK).t()
    q, scales = _to_8_bits(gate / (1.0 + torch.exp(-gate)) * up)
    return {"values": q, "scales": scales}


def _framework(s):
    from logssms_b200.ops import kernels as K
    op = s["op"]
    if op == "norm":
        rows, residual = K.add_rmsnorm_fp8(s["x"], s["weight"], s["eps"], s["residual"], other=s["other"],
                                           in_scales=s["in_scales"], out_scale=s["out_scale"], in_place=False)
        return {"values": rows.values, "scales": rows.scales, "residual": residual}
    if op == "quantize":
        made = (K.quantize_rows_fp8 if s["block_rows"] == 1 else K.quantize_weight_fp8)(s["x"])
        return {"values": made.values, "scales": made.scales}
    x = K.Fp8Rows(s["x"], s["x_scales"])
    if op == "linear":
        return {"y": K.linear_fp8(x, K.Fp8Weight(s["w"], s["w_scales"], settled=True), s["bias"], out_scale=s["out_scale"],
                                  out_dtype=s["dtype"])}
    rows = K.linear_swiglu_fp8(x, K.Fp8Weight(s["gate"], s["gate_scales"], settled=True),
                               K.Fp8Weight(s["up"], s["up_scales"], settled=True), s["act_scale"])
    return {"values": rows.values, "scales": rows.scales}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, rows, width = case["op"], case["rows"], case["width"]
    kb = -(-width // BLOCK)
    if op == "norm":
        size = 2 if case["dtype"] == "bfloat16" else 4
        streams = 2 + case["other"] + case["residual"]                    # read x [, other, residual]; written: the new residual
        return {"bytes": rows * (width * (size * streams + 1) + 4 * kb) + 4 * width, "flops": 8 * rows * width}
    if op == "quantize":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": rows * width * (size + 1) + 4 * kb * -(-rows // case["block_rows"]), "flops": 3 * rows * width}
    features = case["features"]
    fb = -(-features // BLOCK)
    x = rows * (width + 4 * kb)
    if op == "linear":
        out = rows * features * (2 if case["dtype"] == "bfloat16" else 4) + (4 * features if case["bias"] else 0)
        return {"bytes": x + features * width + 4 * fb * kb + out, "flops": 2 * rows * features * width}
    return {"bytes": x + 2 * (features * width + 4 * fb * kb) + rows * (features + 4 * fb), "flops": 4 * rows * features * width}


# ------------------------------------------------------------------ the same in 64 bits
def _in_8_bits(v, block_rows):
    """What the 8-bit values stand for before they are rounded to 8 bits, and their scales, block column by block column."""
    q, scales = torch.empty_like(v), []
    for k in range(0, v.shape[1], BLOCK):
        part = v[:, k:k + BLOCK]
        top = torch.stack([p.abs().max() for p in part.split(block_rows)]) if block_rows > 1 else part.abs().max(1).values
        top = torch.maximum(top / 448, torch.full_like(top, 2.0 ** -126))
        each = top.repeat_interleave(block_rows)[:v.shape[0]]
        q[:, k:k + BLOCK] = part / each.unsqueeze(1)
        scales.append(top)
    return q, torch.stack(scales, 1)


def _product(x, xs, w, ws):
    """Sum over the column blocks of their plain products, each times its two scales."""
    x, w, y = x.double(), w.double(), 0.0
    feature_block = torch.arange(w.shape[0], device=w.device) // BLOCK
    for b, k in enumerate(range(0, x.shape[1], BLOCK)):
        part = torch.mm(x[:, k:k + BLOCK], w[:, k:k + BLOCK].t())
        y = y + part.mul_(xs[:, b].double().unsqueeze(1)).mul_(ws[:, b].double()[feature_block])
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        total = s["in_scales"][0] * s["x"].double()
        for name, factor in (("other", s["in_scales"][1]), ("residual", 1.0)):
            if s[name] is not None:
                total += factor * s[name].double()
        root = torch.sqrt(total.square().sum(1) / case["width"] + s["eps"])
        q, scales = _in_8_bits(total / root.unsqueeze(1) * s["weight"].double() * s["out_scale"], 1)
        return {"values": q, "scales": scales, "residual": total}
    if op == "quantize":
        q, scales = _in_8_bits(s["x"].double(), s["block_rows"])
        return {"values": q, "scales": scales}
    if op == "linear":
        y = _product(s["x"], s["x_scales"], s["w"], s["w_scales"])
        if s["bias"] is not None:
            y = y + s["bias"].double()
        return {"y": y * s["out_scale"]}
    gate = _product(s["x"], s["x_scales"], s["gate"], s["gate_scales"]) * s["act_scale"]
    h = torch.sigmoid(gate).mul_(gate).mul_(_product(s["x"], s["x_scales"], s["up"], s["up_scales"]))
    q, scales = _in_8_bits(h, 1)
    return {"values": q, "scales": scales}
