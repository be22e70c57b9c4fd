"""The MXFP4 operators: quantisation of rows, the dense product, the product
grouped by expert and the routed MoE step on MXFP4 experts.

MXFP4 (OCP Microscaling Formats): blocks of 32 values along the contracted
dimension, each value an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives; two codes a byte, the even element in the low nibble) times one
e8m0 scale (2 ** (code - 127)) a block.  A block's scale is
2 ** (floor(log2(amax)) - 2); its values are rounded to the nearest code, ties
to the even code, magnitudes above 6 to 6.

Kinds (``case["kind"]``):

``quantise``  rows to codes and scales and back to the values they stand for:
              what rounding a tensor to MXFP4 costs, and what it leaves.
``linear``    bf16 rows, quantised, times one MXFP4 weight matrix -> bf16.
``grouped``   the same with rows grouped by expert (ragged boundaries), each
              group times its own expert's matrix; rows of no group give zeros.
``moe``       routed SwiGLU experts: gate and up product of each routed row,
              silu(gate) * up quantised again, down product, sum over the
              row's ranks weighted by its routing weights -> bf16.

The plain forms compute in 32 bits on the dequantised values; the experts'
products are one padded batch each.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, kind, rows, **more):
    case = {"kind": kind, "rows": rows, **more}
    if name is not None:
        case["name"] = name
    return case


def _quantise(name, rows, width, dtype="bfloat16"):
    return _case(name, "quantise", rows, width=width, dtype=dtype)


def _linear(name, rows, k, n):
    return _case(name, "linear", rows, k=k, n=n)


def _grouped(name, rows, experts, k, n, spare=0, skew=False):
    return _case(name, "grouped", rows, experts=experts, k=k, n=n, spare=spare, skew=skew)


def _moe(name, rows, experts, hidden, inter, top_k=8, skew=False):
    return _case(name, "moe", rows, experts=experts, hidden=hidden, inter=inter, top_k=top_k,
                 skew=skew)


def listed():
    return [
        # One token's hidden row, the smallest call there is.
        _quantise("quantise_1x2048", 1, 2048),
        # The rows of a packed prefill of 16 prompts.
        _quantise("quantise_3668x2048", 3668, 2048),
        # A weight tensor at load time: the down matrices of 64 experts, dequantised to fp32.
        _quantise("quantise_131072x768_f32", 131072, 768, "float32"),
        # The packed input projection of one layer (shared gate and up rows,
        # 256 router rows, the shared expert's gate: an odd width), one token.
        _linear("linear_1_k2048_n1281", 1, 2048, 1281),
        # The same projection for a full decode bucket that is three quarters live.
        _linear("linear_52_k2048_n1281", 52, 2048, 1281),
        # The same projection over the largest prefill capacity in use.
        _linear("linear_4096_k2048_n1281", 4096, 2048, 1281),
        # A wide square projection over twice those rows, one short.
        _linear("linear_8191_k4096_n4096", 8191, 4096, 4096),
        # Gate and up matrices of 128 experts for the routes of 48 live decode slots.
        _grouped("grouped_384_e128", 384, 128, 2048, 1536),
        # The reference model's gate and up matrices over the routes of 2048
        # prompt rows, in a buffer with spare rows after the last group.
        _grouped("grouped_16384_e256", 16384, 256, 2048, 1024, spare=609, skew=True),
        # One token through the reference model's routed experts.
        _moe("moe_1_e256", 1, 256, 2048, 512),
        # A full decode bucket of the reference model.
        _moe("moe_64_e256", 64, 256, 2048, 512),
        # The packed prefill of 16 prompts over 128 experts of uneven popularity.
        _moe("moe_3668_e128", 3668, 128, 2048, 768, skew=True),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "grouped", "grouped", "moe", "moe", "moe"])
    if kind == "quantise":
        width = BLOCK * _spread(rng, 1, 256)
        rows = _spread(rng, 1, 100_000_000 // width)
        return _quantise(None, rows, width, rng.choice(["bfloat16", "float32"]))
    if kind == "linear":
        return _linear(None, _spread(rng, 1, 8191), 128 * rng.randint(1, 32), _spread(rng, 16, 4096))
    if kind == "grouped":
        return _grouped(None, _spread(rng, 1, 16384), rng.choice([1, 7, 16, 60, 128, 256]),
                        128 * rng.randint(1, 16), _spread(rng, 32, 2048),
                        spare=rng.choice([0, 0, _spread(rng, 1, 512)]), skew=rng.random() < 0.4)
    skew = rng.random() < 0.4
    shape = rng.choice([(16, 1024, 256), (128, 2048, 768), (256, 2048, 512), None])
    if shape is None:
        shape = (rng.choice([8, 60, 200]), 128 * rng.randint(2, 16), 128 * rng.randint(1, 6))
    return _moe(None, _spread(rng, 1, 3668), *shape, top_k=rng.choice([8, 8, 8, 4, 2, 1]), skew=skew)


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _blocks(x):
    """fp32 [..., K] -> (e2m1 codes uint8 [..., K], e8m0 codes int32 [..., K / 32])."""
    v = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    _, exponent = torch.frexp(amax)  # amax = m * 2 ** exponent, m in [0.5, 1)
    shift = (exponent - 3).clamp(-127, 127)
    shift = torch.where(amax > 0, shift, torch.full_like(shift, -127))
    a = torch.ldexp(v.abs(), -shift)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    code = code + 8 * (v < 0).to(torch.uint8)
    return code.reshape(x.shape), (shift + 127).squeeze(-1)


def _values(code, scale_code):
    """e2m1 codes [..., K] and e8m0 codes [..., K / 32] -> fp32 values [..., K]."""
    table = torch.tensor(GRID + tuple(-g for g in GRID), device=code.device)
    v = table[code.to(torch.int32)].reshape(*scale_code.shape, BLOCK)
    return torch.ldexp(v, scale_code.to(torch.int32).unsqueeze(-1) - 127).reshape(code.shape)


def _rounded(x):
    return _values(*_blocks(x))


def _unpacked(codes):
    return torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)


def _weights(packed):
    codes, scales = packed
    return _values(_unpacked(codes), scales)


def _padded(group, position, most, groups, rows):
    """Rows of each group in a [groups, most, K] batch, zeros behind them."""
    batch = torch.zeros(groups, most, rows.shape[-1], device=rows.device)
    batch[group, position] = rows
    return batch


def _by_group(group, groups):
    """Each entry's position in its group, in order."""
    order = torch.argsort(group, stable=True)
    counts = torch.zeros(groups, dtype=torch.int64, device=group.device)
    counts.scatter_add_(0, group, torch.ones_like(group))
    first = counts.cumsum(0) - counts
    position = torch.empty_like(order)
    position[order] = torch.arange(len(group), device=group.device) - first[group[order]]
    return position


def _plain_quantise(state):
    code, scale = _blocks(state["x"].float())
    return _values(code, scale).to(torch.bfloat16), scale.to(torch.uint8)


def _plain_linear(state):
    return (_rounded(state["x"].float()) @ _weights(state["w"]).T).to(torch.bfloat16)


def _plain_grouped(state):
    x, bounds, groups = _rounded(state["x"].float()), state["boundaries"].long(), state["groups"]
    row = torch.arange(len(x), device=x.device)
    group = torch.searchsorted(bounds, row, right=True) - 1
    live = (group >= 0) & (group < groups)
    group = group.clamp(0, groups - 1)
    position = torch.where(live, row - bounds[group], state["most"])  # rows of no group: a spare slot
    batch = _padded(group, position, state["most"] + 1, groups, x)
    y = torch.bmm(batch, _weights(state["w"]).transpose(1, 2))[group, position]
    return torch.where(live[:, None], y, 0.0).to(torch.bfloat16)


def _plain_moe(state):
    x, ids, experts = _rounded(state["x"].float()), state["ids"], state["groups"]
    rows, top_k = ids.shape
    expert = ids.reshape(-1)
    position = _by_group(expert, experts)
    batch = _padded(expert, position, state["most"], experts, x.repeat_interleave(top_k, 0))
    gate, up = torch.bmm(batch, _weights(state["w13"]).transpose(1, 2)).chunk(2, -1)
    act = _rounded(gate / (1 + torch.exp(-gate)) * up)
    down = torch.bmm(act, _weights(state["w2"]).transpose(1, 2))[expert, position]
    return (down.reshape(rows, top_k, -1) * state["weights"].float()[..., None]).sum(1).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _package():
    path = str(Path(__file__).resolve().parents[1] / "drama-3-single-b300-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from drama3_amd import mxfp4

    return mxfp4


def _own_quantise(state):
    mx = _package()
    codes, scales = mx.quantize_mxfp4(state["x"])
    return mx.dequantize_mxfp4(codes, scales), scales


def _own_linear(state):
    return _package().mxfp4_linear(state["x"], state["handle"])


def _own_grouped(state):
    return _package().grouped_mxfp4(state["x"], state["boundaries"], state["handle"])


def _own_moe(state):
    return _package().mxfp4_moe(state["x"], state["ids"], state["weights"], state["handle"])


# ---------------------------------------------------------------------------
def _random_rows(gen, rows, width):
    """Hidden rows: normal values, rows of different size, a few large channels."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return x * torch.exp(0.4 * torch.randn(width, generator=gen, device="cuda"))


def _random_weight(gen, *shape):
    w = torch.randn(*shape, generator=gen, device="cuda") * shape[-1] ** -0.5
    w *= torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    code, scale = _blocks(w)
    return (code[..., 0::2] | code[..., 1::2] << 4).contiguous(), scale.to(torch.uint8)


def _random_logits(gen, rows, experts, skew):
    logits = torch.randn(rows, experts, generator=gen, device="cuda")
    if skew:  # some experts are chosen far more often than others
        logits = logits + 0.75 * torch.randn(experts, generator=gen, device="cuda")
    return logits


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    kind, rows = case["kind"], case["rows"]
    state = {"kind": kind}
    if kind == "quantise":
        state["x"] = _random_rows(gen, rows, case["width"]).to(getattr(torch, case["dtype"]))
    elif kind == "linear":
        state["x"] = _random_rows(gen, rows, case["k"]).to(torch.bfloat16)
        state["w"] = _random_weight(gen, case["n"], case["k"])
        if own:
            state["handle"] = _package().prepare_mxfp4(*state["w"])
    elif kind == "grouped":
        experts = case["experts"]
        state["x"] = _random_rows(gen, rows + case["spare"], case["k"]).to(torch.bfloat16)
        state["w"] = _random_weight(gen, experts, case["n"], case["k"])
        chosen = _random_logits(gen, rows, experts, case["skew"]).argmax(-1)
        counts = torch.bincount(chosen, minlength=experts)
        state["boundaries"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        state["groups"], state["most"] = experts, int(counts.max())
        if own:
            state["handle"] = _package().prepare_mxfp4(*state["w"])
    else:
        experts, hidden, inter = case["experts"], case["hidden"], case["inter"]
        state["x"] = _random_rows(gen, rows, hidden).to(torch.bfloat16)
        state["w13"] = _random_weight(gen, experts, 2 * inter, hidden)
        state["w2"] = _random_weight(gen, experts, hidden, inter)
        top, ids = _random_logits(gen, rows, experts, case["skew"]).topk(case["top_k"], -1)
        state["ids"], state["weights"] = ids, top.softmax(-1).to(torch.bfloat16)
        state["groups"] = experts
        state["most"] = int(torch.bincount(ids.reshape(-1), minlength=experts).max())
        if own:
            state["handle"] = _package().prepare_mxfp4_experts(*state["w13"], *state["w2"])
    return state


def run(state):
    if own:
        return {"quantise": _own_quantise, "linear": _own_linear, "grouped": _own_grouped,
                "moe": _own_moe}[state["kind"]](state)
    return {"quantise": _plain_quantise, "linear": _plain_linear, "grouped": _plain_grouped,
            "moe": _plain_moe}[state["kind"]](state)


def _used(experts, choices):
    """How many of the experts that many choices reach on average."""
    return experts * (1.0 - (1.0 - 1.0 / experts) ** choices)


def _weight_bytes(count):
    return count / 2 + count / BLOCK


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "quantise":
        count = rows * case["width"]
        size = 4 if case["dtype"] == "float32" else 2
        # read once; the values and the scales written.  A maximum, a product
        # and a rounding an element, and a product on the way back.
        return {"bytes": count * (size + 2) + count // BLOCK, "flops": 4 * count}
    if kind == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": rows * (k + n) * 2 + _weight_bytes(n * k), "flops": 2 * rows * n * k}
    if kind == "grouped":
        k, n = case["k"], case["n"]
        return {"bytes": rows * (k + n) * 2 + case["spare"] * n * 2
                + _weight_bytes(_used(case["experts"], rows) * n * k), "flops": 2 * rows * n * k}
    hidden, inter, pairs = case["hidden"], case["inter"], rows * case["top_k"]
    weight = 3 * hidden * inter
    return {"bytes": rows * hidden * 4 + pairs * 10 + _weight_bytes(_used(case["experts"], pairs) * weight),
            "flops": 2 * pairs * weight}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_blocks(x):
    """fp64 [..., K] -> (values, e8m0 codes): every value rounded, half to
    even, to a multiple of the step of its binade."""
    v = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    top = v.abs().max(-1, keepdim=True).values
    power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    power = power + (torch.exp2(power + 1) <= top).double() - (torch.exp2(power) > top).double()
    power = torch.where(top > 0, power - 2, -127.0).clamp(-127, 127)
    scale = torch.exp2(power)
    v = v / scale
    mag = v.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    v = torch.sign(v) * (torch.round(mag / step) * step).clamp(max=6.0)
    return (v * scale).reshape(x.shape), (power + 127).squeeze(-1)


def _exact_weights(packed):
    codes, scales = packed
    nibbles = torch.empty(*codes.shape, 2, dtype=torch.int16, device=codes.device)
    nibbles[..., 0], nibbles[..., 1] = codes % 16, codes // 16
    exponent, mantissa = (nibbles // 2) % 4, nibbles % 2
    mag = torch.where(exponent == 0, mantissa * 0.5,
                      torch.exp2(exponent.double() - 1) * (1 + 0.5 * mantissa.double()))
    value = torch.where(nibbles < 8, mag, -mag).reshape(*codes.shape[:-1], -1)
    scale = torch.exp2(scales.double() - 127)
    return value * scale.repeat_interleave(BLOCK, -1)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        values, scale = _exact_blocks(state["x"].double())
        return values, scale.to(torch.uint8)
    x, _ = _exact_blocks(state["x"].double())
    if kind == "linear":
        return x @ _exact_weights(state["w"]).T
    if kind == "grouped":
        ends = state["boundaries"].tolist()
        out = torch.zeros(len(x), case["n"], dtype=torch.float64, device=x.device)
        codes, scales = state["w"]
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            if b > a:
                out[a:b] = x[a:b] @ _exact_weights((codes[e], scales[e])).T
        return out
    ids, weights = state["ids"], state["weights"].double()
    out = torch.zeros(len(x), case["hidden"], dtype=torch.float64, device=x.device)
    for e in torch.unique(ids).tolist():
        row, rank = torch.nonzero(ids == e, as_tuple=True)
        both = x[row] @ _exact_weights((state["w13"][0][e], state["w13"][1][e])).T
        gate, up = both[:, :case["inter"]], both[:, case["inter"]:]
        act, _ = _exact_blocks(gate * torch.sigmoid(gate) * up)
        y = act @ _exact_weights((state["w2"][0][e], state["w2"][1][e])).T
        out.index_add_(0, row, y * weights[row, rank][:, None])
    return out
