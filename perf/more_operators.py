"""The operators of 4-bit weights whose speed is measured, over the sizes, data types and
row counts they are used at: the product with weights held in 4 bits, its gated form, the
residual norm that gives 8-bit rows, a feed-forward block of them, and the packing.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is one pass: the
operators in plain torch, or with ``own`` the calls that a program makes of
``qdc_amd.quant_ops``.  ``exact`` is the same result in 64 bits from the definition.

A weight ``[out, inner]`` is a whole number of -8..7 times the bf16 scale of its group of
``group`` inputs; a model keeps it as blocks of 16 outputs by 128 inputs (``_blocks``).
8-bit rows are whole numbers of -127..127 times the fp32 scale of their group of 128
columns.  What is held in 4 or 8 bits is returned as the values it stands for.
"""
import math
import os
import sys

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUPS = (32, 64, 128)
Q8_GROUP = 128


def _framework():
    """The framework's operators, imported at the first call and not at each."""
    ops = sys.modules.get("qdc_amd.quant_ops")
    if ops is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                               "qwendecisioncore.jl_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from qdc_amd import quant_ops as ops
    return ops


# -------------------------------------------------------------------- cases --
def listed():
    return [
        # The small decision model scoring one more token: a launch and its latency.
        _linear("linear_1x256x768_f32", 1, 256, 768, 32, "f32", "f32"),
        # One token through an attention layer's q, k, v and gate projection.
        _linear("linear_1x1024x5120_bf16", 1, 1024, 5120, 64, "bf16", "bf16"),
        # A step of a batch: the feed-forward block's way back into the residual stream.
        _linear("linear_24x3584x1024_bf16", 24, 3584, 1024, 128, "bf16", "f32"),
        # A short odd prompt of a wider model kept in fp32.
        _linear("linear_301x2048x6144_f32", 301, 2048, 6144, 32, "f32", "f32"),
        # Eight prompts of 2048 tokens through a linear attention layer's projection.
        _linear("linear_16384x1024x8224_q8", 16384, 1024, 8224, 64, "q8", "bf16"),
        # One token's gate and up projections, and the same of eight prompts.
        _gated("gated_1x1024x3584_bf16", 1, 1024, 3584, 64, "bf16", "bf16"),
        _gated("gated_16384x1024x3584_q8", 16384, 1024, 3584, 64, "q8", "q8"),
        # A feed-forward block of a batch's step, norm to down projection.
        {"name": "block_77x1024x3584", "kind": "block", "rows": 77, "inner": 1024,
         "inter": 3584, "group": 64},
        # The norm of one token, and of eight padded prompts.
        _norm("norm_1x1024", 1, 1024, "bf16", 0.0),
        _norm("norm_16384x1024", 16384, 1024, "bf16", 0.15),
        # A layer's gate and up weights as a checkpoint has them, and an odd fp32 one.
        _pack("pack_7168x1024_bf16", 7168, 1024, 64, "bf16"),
        _pack("pack_1011x2120_f32", 1011, 2120, 32, "f32"),
    ]


def _linear(name, rows, inner, out, group, x, dtype):
    return {"name": name, "kind": "linear", "rows": rows, "inner": inner, "out": out,
            "group": group, "x": x, "dtype": dtype}


def _gated(name, rows, inner, inter, group, x, dtype):
    return {"name": name, "kind": "gated", "rows": rows, "inner": inner, "inter": inter,
            "group": group, "x": x, "dtype": dtype}


def _norm(name, rows, width, dtype, masked):
    """``masked``: the share of rows that are padding."""
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype,
            "masked": masked}


def _pack(name, out, inner, group, dtype):
    return {"name": name, "kind": "pack", "out": out, "inner": inner, "group": group,
            "dtype": dtype}


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gated", "gated", "block", "norm", "pack"])
    group = rng.choice(GROUPS)
    if kind == "norm":
        width = 16 * _log_int(rng, 4, 512)
        case = _norm("", _log_int(rng, 1, 16384 * 1024 // max(1024, width)), width,
                     rng.choice(["f32", "bf16"]), rng.choice([0.0, 0.2]))
    elif kind == "pack":
        case = _pack("", _log_int(rng, 1, 8224), 8 * _log_int(rng, 4, 448), group,
                     rng.choice(["f32", "bf16"]))
    else:
        x = rng.choice(["f32", "bf16", "bf16", "q8"])
        inner = 16 * _log_int(rng, 4, 448)
        # fp32 rows are multiplied as three terms
        most = 16384 * 1024 * 7168 // (4 if x == "f32" else 1)
        if kind == "linear":
            out = _log_int(rng, 1, 8224)
            case = _linear("", _log_int(rng, 1, max(1, min(16384, most // (inner * out)))), inner,
                           out, group, x, rng.choice(["f32", "bf16"]))
        elif kind == "gated":
            inter = 16 * _log_int(rng, 1, 384) if rng.random() < 0.7 else _log_int(rng, 1, 6144)
            case = _gated("", _log_int(rng, 1, max(1, min(16384, most // (2 * inner * inter)))),
                          inner, inter, group, x,
                          rng.choice(["f32", "bf16", "q8"] if inter % 16 == 0 else ["f32", "bf16"]))
        else:
            inner, inter = 16 * _log_int(rng, 4, 128), 16 * _log_int(rng, 4, 384)
            case = {"kind": "block", "rows": _log_int(rng, 1, min(4096, most // (3 * inner * inter))),
                    "inner": inner, "inter": inter, "group": group}
    case.pop("name", None)
    return case


# ------------------------------------------------------------------- inputs --
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _rows(g, rows, width):
    """Rows as they leave a norm: of unit size, a few columns far larger."""
    x = _randn(g, rows, width)
    x[:, torch.randint(width, (max(1, width // 200),), generator=g, device=DEVICE)] *= 8
    return x


def _weight(g, out, inner, group):
    """Whole numbers ``[out, inner]`` (int8) and scales ``[out, groups]`` (bf16)."""
    ints = (_randn(g, out, inner) * 2.6).round().clamp(-7, 7).to(torch.int8)
    scales = (0.008 * (1.0 + 0.2 * _randn(g, out, -(-inner // group)).clamp(-3, 3))).to(torch.bfloat16)
    return ints, scales


def _blocks(ints, scales, group, gated=False):
    """The form a model keeps: 16 outputs x 128 inputs a block of 64 lanes x 4 words, word t
    of lane l the inputs 32 t + 8 (l // 16) + 0..7 of output l % 16, input j < 4 in bits
    8 j .. 8 j + 3 and input 4 + j above it; scales [block, group, output].  Zeros behind
    the last output and input; gated: a block of gate, then one of up, in turn."""
    out, inner = ints.shape
    if gated:
        both = (_blocks(i, s, group) for i, s in zip(ints.chunk(2), scales.chunk(2)))
        return tuple(torch.stack(p, 1).flatten(0, 1).contiguous() for p in zip(*both))
    nb, kb = -(-out // 16), -(-inner // 128)
    q = ints.new_zeros((nb * 16, kb * 128))
    q[:out, :inner] = ints & 15
    q = q.view(nb, 16, kb, 4, 4, 2, 4).int()              # n, k: t, quarter, upper, j
    byte = q[..., 0, :] | q[..., 1, :] << 4
    words = byte.to(torch.uint8).permute(0, 2, 4, 1, 3, 5).contiguous().view(torch.int32)
    sc = scales.new_zeros((nb * 16, kb * 128 // group))
    sc[:out, :scales.shape[1]] = scales
    return words.view(nb, kb, 64, 4), sc.view(nb, 16, -1).transpose(1, 2).contiguous()


def _q8_rows(g, rows, width):
    scales = 0.02 + 0.02 * torch.rand((rows, -(-width // Q8_GROUP)), generator=g, device=DEVICE)
    return (_randn(g, rows, width) * 40).round().clamp(-127, 127).to(torch.int8), scales


def _prepare_linear(case, g, gated=False):
    rows, inner = case["rows"], case["inner"]
    out = 2 * case["inter"] if gated else case["out"]
    ints, scales = _weight(g, out, inner, case["group"])
    x = _q8_rows(g, rows, inner) if case["x"] == "q8" else \
        _rows(g, rows, inner).to(TYPES[case["x"]])
    return {"x": x, "ints": ints, "scales": scales,
            "packed": _blocks(ints, scales, case["group"], gated)}


def _prepare_norm(case, g):
    rows, width = case["rows"], case["width"]
    mask = None
    if case["masked"]:
        mask = (torch.rand(rows, generator=g, device=DEVICE) >= case["masked"]).int()
    return {"x": _rows(g, rows, width), "add": _randn(g, rows, width), "mask": mask,
            "weight": (_randn(g, width) * 0.1).to(TYPES[case["dtype"]])}


def _prepare_block(case, g):
    norm = _prepare_norm({"rows": case["rows"], "width": case["inner"], "masked": 0.0,
                          "dtype": "bf16"}, g)
    up = _weight(g, 2 * case["inter"], case["inner"], case["group"])
    down = _weight(g, case["inner"], case["inter"], case["group"])
    return norm | {"up": up, "down": down, "up_packed": _blocks(*up, case["group"], True),
                   "down_packed": _blocks(*down, case["group"])}


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind in ("linear", "gated"):
        state = _prepare_linear(case, g, kind == "gated")
    elif kind == "norm":
        state = _prepare_norm(case, g)
    elif kind == "block":
        state = _prepare_block(case, g)
    else:
        state = {"w": (_randn(g, case["out"], case["inner"]) * 0.02).to(TYPES[case["dtype"]])}
    return state | {"case": case}


# ---------------------------------------------------------------------- run --
def run(state):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


def _own_x(qo, s):
    return qo.Q8(*s["x"]) if s["case"]["x"] == "q8" else s["x"]


def _own_linear(s):
    qo, c = _framework(), s["case"]
    w = qo.W4(*s["packed"], c["out"], c["inner"], c["group"], False)
    return qo.linear_w4(_own_x(qo, s), w, out_dtype=TYPES[c["dtype"]])


def _own_gated(s):
    qo, c = _framework(), s["case"]
    w = qo.W4(*s["packed"], 2 * c["inter"], c["inner"], c["group"], True)
    if c["dtype"] == "q8":
        return qo.dequantize_q8(qo.gated_w4(_own_x(qo, s), w, out_dtype=qo.Q8), torch.bfloat16)
    return qo.gated_w4(_own_x(qo, s), w, out_dtype=TYPES[c["dtype"]])


def _own_norm(s):
    qo = _framework()
    residual, rows = qo.residual_rms_q8(s["x"], s["add"], s["weight"], EPS, token_mask=s["mask"])
    return residual, qo.dequantize_q8(rows, torch.bfloat16)


def _own_block(s):
    qo, c = _framework(), s["case"]
    up = qo.W4(*s["up_packed"], 2 * c["inter"], c["inner"], c["group"], True)
    down = qo.W4(*s["down_packed"], c["inner"], c["inter"], c["group"], False)
    residual, rows = qo.residual_rms_q8(s["x"], s["add"], s["weight"], EPS)
    act = qo.gated_w4(rows, up, out_dtype=qo.Q8)
    return residual, qo.linear_w4(act, down, out_dtype=torch.bfloat16)


def _own_pack(s):
    qo = _framework()
    return qo.unpack_w4(qo.pack_w4(s["w"], group=s["case"]["group"]), torch.float32)


_OWN = {"linear": _own_linear, "gated": _own_gated, "norm": _own_norm, "block": _own_block,
        "pack": _own_pack}


# -------------------------------------------------------------- plain forms --
def _spread(values, scales, group):
    """``values * scales`` with a scale for each ``group`` columns, in 32 bits."""
    wide = scales.float().repeat_interleave(group, 1)[:, :values.shape[1]]
    return values.float() * wide


def _plain_x(s):
    return _spread(*s["x"], Q8_GROUP) if s["case"]["x"] == "q8" else s["x"].float()


def _plain_q8(v):
    """The values that 8 bits hold of ``v``, in 32 bits."""
    width = v.shape[1]
    v = torch.nn.functional.pad(v, (0, -width % Q8_GROUP)).view(v.shape[0], -1, Q8_GROUP)
    scale = v.abs().amax(-1, keepdim=True) / 127.0
    q = torch.where(scale > 0, v / scale, 0.0).round().clamp(-127, 127)
    return (q * scale).flatten(1)[:, :width]


def _plain_linear(s):
    w = _spread(s["ints"], s["scales"], s["case"]["group"])
    return (_plain_x(s) @ w.t()).to(TYPES[s["case"]["dtype"]])


def _plain_act(x, weight, group):
    gate, up = (x @ _spread(*weight, group).t()).chunk(2, 1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_gated(s):
    act = _plain_act(_plain_x(s), (s["ints"], s["scales"]), s["case"]["group"])
    if s["case"]["dtype"] == "q8":
        return _plain_q8(act).bfloat16()
    return act.to(TYPES[s["case"]["dtype"]])


def _plain_rms(s):
    residual = s["x"] + s["add"]
    normed = residual * torch.rsqrt(residual.square().mean(1, keepdim=True) + EPS)
    normed = normed * (1.0 + s["weight"].float())
    if s["mask"] is not None:
        normed = torch.where(s["mask"][:, None] != 0, normed, 0.0)
    return residual, _plain_q8(normed)


def _plain_norm(s):
    residual, values = _plain_rms(s)
    return residual, values.bfloat16()


def _plain_block(s):
    group = s["case"]["group"]
    residual, x = _plain_rms(s)
    act = _plain_q8(_plain_act(x, s["up"], group))
    return residual, (act @ _spread(*s["down"], group).t()).bfloat16()


def _plain_pack(s):
    group = s["case"]["group"]
    out, inner = s["w"].shape
    w = torch.nn.functional.pad(s["w"].float(), (0, -inner % group)).view(out, -1, group)
    # quotients in 64 bits, as one next to a half would be rounded to it in 32
    scale = (w.abs().amax(-1, keepdim=True).double() / 7.0).bfloat16().float()
    q = torch.where(scale > 0, w.double() / scale.double(), 0.0).round().clamp(-7, 7)
    return (q.float() * scale).flatten(1)[:, :inner].contiguous()


_PLAIN = {"linear": _plain_linear, "gated": _plain_gated, "norm": _plain_norm,
          "block": _plain_block, "pack": _plain_pack}


# --------------------------------------------------------------- yardsticks --
def work(case):
    size = {"f32": 4, "bf16": 2, "q8": 1 + 4 / Q8_GROUP}
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["width"]
        # x and add read, the residual and the 8-bit rows written
        return {"bytes": n * (12 + size["q8"]), "flops": 10 * n}
    weight = lambda out, inner: out * inner // 2 + 2 * out * -(-inner // case["group"])  # noqa: E731
    if kind == "pack":
        out, inner = case["out"], case["inner"]
        return {"bytes": out * inner * size[case["dtype"]] + weight(out, inner),
                "flops": 4 * out * inner}
    rows, inner = case["rows"], case["inner"]
    if kind == "block":
        inter = case["inter"]
        return {"bytes": weight(2 * inter, inner) + weight(inner, inter) + rows * inner * (12 + 2),
                "flops": 6 * rows * inner * inter}
    out = case["out"] if kind == "linear" else 2 * case["inter"]
    written = rows * (out if kind == "linear" else case["inter"]) * size[case["dtype"]]
    return {"bytes": weight(out, inner) + rows * inner * size[case["x"]] + written,
            "flops": 2 * rows * out * inner}


# ---------------------------------------------------------- 64-bit reference --
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


def _times(ints, scales, group):
    """The numbers that whole numbers and the scales of their groups stand for."""
    column = torch.arange(ints.shape[1], device=DEVICE)
    return ints.double() * scales.double()[:, column // group]


def _exact_q8(v):
    width = v.shape[1]
    out = torch.empty_like(v)
    for first in range(0, width, Q8_GROUP):
        part = v[:, first:first + Q8_GROUP]
        step = part.abs().max(1, keepdim=True).values / 127
        whole = torch.round(part / torch.where(step == 0, 1.0, step))
        out[:, first:first + Q8_GROUP] = whole * step
    return out


def _exact_x(s):
    return _times(*s["x"], Q8_GROUP) if s["case"]["x"] == "q8" else s["x"].double()


def _exact_linear(s):
    return torch.mm(_exact_x(s), _times(s["ints"], s["scales"], s["case"]["group"]).t())


def _exact_silu(x, weight, group):
    both = torch.mm(x, _times(*weight, group).t())
    half = both.shape[1] // 2
    return both[:, :half] * torch.sigmoid(both[:, :half]) * both[:, half:]


def _exact_gated(s):
    act = _exact_silu(_exact_x(s), (s["ints"], s["scales"]), s["case"]["group"])
    return _exact_q8(act) if s["case"]["dtype"] == "q8" else act


def _exact_norm(s):
    residual = s["x"].double() + s["add"].double()
    size = torch.sqrt((residual ** 2).sum(1, keepdim=True) / residual.shape[1] + EPS)
    normed = residual / size * (s["weight"].double() + 1)
    if s["mask"] is not None:
        normed = normed.masked_fill(s["mask"][:, None] == 0, 0.0)
    return residual, _exact_q8(normed)


def _exact_block(s):
    group = s["case"]["group"]
    residual, x = _exact_norm(s)
    act = _exact_q8(_exact_silu(x, s["up"], group))
    return residual, torch.mm(act, _times(*s["down"], group).t())


def _exact_pack(s):
    group, w = s["case"]["group"], s["w"].double()
    out = torch.empty_like(w)
    for first in range(0, w.shape[1], group):
        part = w[:, first:first + group]
        # the scale is held in bf16
        step = (part.abs().max(1, keepdim=True).values / 7).bfloat16().double()
        whole = torch.round(part / torch.where(step == 0, 1.0, step)).clamp(-7, 7)
        out[:, first:first + group] = whole * step
    return out


_EXACT = {"linear": _exact_linear, "gated": _exact_gated, "norm": _exact_norm,
          "block": _exact_block, "pack": _exact_pack}
