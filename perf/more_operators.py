"""The attention operators over packed rows and a paged cache: rotary positions,
appending keys and values to the cache with the rotation on the way, and the
attention of new tokens over the cached ones.

Kinds (``case["kind"]``):

``rope``    rotates rows [T, H, D] by their positions: pair (a, b) at frequency
            f becomes (a cos - b sin, a sin + b cos) * magnitude at the angle
            position * f.  Half layout: pairs (i, i + R / 2) of the first R
            columns; interleaved: (2 i, 2 i + 1); columns from R on stay.
            f_i = base ** (-2 i / R), scaled for long contexts by ``scaling``:
            "linear" f / s; "base" base * s ** (R / (R - 2)) as the base;
            "bands" w f + (1 - w) f / s with w = clamp((r - 1) / 31, 0, 1) for
            r = original * f / (2 pi) turns, and magnitude 0.1 ln s + 1.
``append``  rotates the queries and keys of new tokens and writes keys and
            values to their place: page ``page_table[slot, position // P]``,
            token ``position % P`` of [pages, kv heads, P, D], in bf16 or in
            e4m3 (value / the head's scale, clamped to +-448).  Rows of a
            negative slot or position and of unmapped pages (-1) go nowhere.
``attend``  rows [b_i, b_{i+1}) are the n_i newest tokens of sequence i, which
            has L_i tokens in the cache.  Row j of it attends the mapped keys up
            to its own position L_i - n_i + j, the last ``window`` of them
            where one is given.  Rows without a key give zeros, and so do rows
            of no sequence.

The plain forms compute in 32 bits (angles and what is rounded to 8 bits in 64)
on padded batches.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

GOLDEN = 0.6180339887498949


def _case(name, kind, **more):
    case = {"kind": kind, **more}
    if name is not None:
        case["name"] = name
    return case


def _rope(name, rows, heads, dim, rotary, interleaved=False, scaling="none", dtype="bfloat16", far=2048):
    return _case(name, "rope", rows=rows, heads=heads, dim=dim, rotary=rotary, interleaved=interleaved,
                 scaling=scaling, dtype=dtype, far=far)


def _append(name, sequences, rows, heads, kv_heads, dim, rotary, page=16, cache="bfloat16", prior=0,
            spare=0, interleaved=False):
    """``rows`` new tokens shared among the sequences, on top of up to ``prior`` cached ones."""
    return _case(name, "append", sequences=sequences, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim,
                 rotary=rotary, page=page, cache=cache, prior=prior, spare=spare, interleaved=interleaved)


def _attend(name, heads, kv_heads, dim, decode=0, context=0, prompts=0, chunk=0, prior=0, page=16,
            cache="bfloat16", window=0, spare=0):
    """``decode`` sequences of one new token and up to ``context`` keys, then
    ``prompts`` of up to ``chunk`` new tokens on top of up to ``prior`` cached ones."""
    return _case(name, "attend", heads=heads, kv_heads=kv_heads, dim=dim, decode=decode, context=context,
                 prompts=prompts, chunk=chunk, prior=prior, page=page, cache=cache, window=window, spare=spare)


def listed():
    return [
        # The queries of one decode token, a quarter of each head rotated.
        _rope("rope_1x16x256", 1, 16, 256, 64),
        # Queries and keys of a packed prefill far into a long context, adjacent pairs.
        _rope("rope_8191x40x128_far", 8191, 40, 128, 128, interleaved=True, scaling="bands", far=131072),
        # A full decode bucket: one new token for each of 64 slots.
        _append("append_64_decode", 64, 64, 16, 2, 256, 64, prior=2047),
        # The packed prefill of 16 prompts from an empty cache, with spare rows behind them.
        _append("append_3668_prompts", 16, 3668, 16, 2, 128, 128, spare=172),
        # Long chunks into an e4m3 cache of larger pages.
        _append("append_8192_e4m3", 4, 8192, 32, 8, 128, 128, page=64, cache="float8_e4m3fn", prior=8192,
                interleaved=True),
        # One token of one short sequence, the smallest step there is.
        _attend("attend_1_short", 16, 2, 128, decode=1, context=333),
        # A decode bucket that is three quarters live, at the longest context in use.
        _attend("attend_52_decode", 16, 2, 256, decode=52, context=2048),
        # Long contexts in an e4m3 cache, few sequences: the keys' bytes alone count.
        _attend("attend_16_long_e4m3", 32, 8, 128, decode=16, context=32768, page=64, cache="float8_e4m3fn"),
        # A mixed step: decode rows first, then prompts, spare rows at the end.
        _attend("attend_mixed", 16, 2, 128, decode=48, context=2048, prompts=4, chunk=401, spare=37),
        # The packed prefill of 16 prompts from an empty cache, heads of their own keys, a sliding window.
        _attend("attend_16_prompts_window", 16, 16, 64, prompts=16, chunk=1024, window=300),
        # A whole long prompt.
        _attend("attend_8192_prompt", 16, 4, 128, prompts=1, chunk=8192, page=32),
        # A chunk of a long prompt on top of what is cached, the largest.
        _attend("attend_4096_chunk", 32, 8, 128, prompts=1, chunk=4096, prior=20480, page=64),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend"])
    if kind == "rope":
        dim = rng.choice([32, 64, 80, 128, 256])
        heads = rng.choice([1, 2, 7, 16, 40])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        rows = _spread(rng, 1, 40_000_000 // (heads * dim) if rng.random() < 0.5 else 4096)
        far = rng.choice([2048, 131072])
        return _rope(None, min(rows, 16384), heads, dim, rotary, rng.random() < 0.5,
                     rng.choice(["none", "linear", "base", "bands"]), rng.choice(["bfloat16", "bfloat16", "float32"]),
                     far)
    dim = rng.choice([64, 128, 128, 256])
    heads, kv_heads = rng.choice([(16, 2), (32, 8), (16, 4), (8, 8), (12, 4), (20, 4), (9, 1), (24, 1)])
    page = rng.choice([16, 16, 32, 64, 128])
    cache = rng.choice(["bfloat16", "bfloat16", "float8_e4m3fn"])
    if kind == "append":
        sequences = _spread(rng, 1, 64)
        rows = max(sequences, _spread(rng, 1, 8192))
        return _append(None, sequences, rows, heads, kv_heads, dim, rng.choice([dim, dim // 2, dim // 4]), page, cache,
                       prior=rng.choice([0, _spread(rng, 1, 4096)]), spare=rng.choice([0, 0, _spread(rng, 1, 200)]),
                       interleaved=rng.random() < 0.5)
    window = rng.choice([0, 0, 0, _spread(rng, 1, 2048)])
    shape = rng.choice(["decode", "decode", "chunk", "mixed"])
    spare = rng.choice([0, 0, _spread(rng, 1, 100)])
    more = dict(page=page, cache=cache, window=window, spare=spare)
    if shape == "decode":
        decode = _spread(rng, 1, 96)
        return _attend(None, heads, kv_heads, dim, decode=decode, context=_spread(rng, 1, min(65536, 400_000 // decode)),
                       **more)
    if shape == "chunk":
        prompts = _spread(rng, 1, 16)
        chunk = _spread(rng, 2, 4096 // prompts)
        return _attend(None, heads, kv_heads, dim, prompts=prompts, chunk=chunk,
                       prior=rng.choice([0, _spread(rng, 1, 16384 // prompts)]), **more)
    return _attend(None, heads, kv_heads, dim, decode=_spread(rng, 1, 60), context=_spread(rng, 1, 2048),
                   prompts=rng.randint(1, 4), chunk=_spread(rng, 2, 600), prior=rng.choice([0, 500]), **more)


# ---------------------------------------------------------------------------
# What the cases' sequences are: the same for every seed, of uneven lengths
# ---------------------------------------------------------------------------
def _sizes(count, most):
    """``count`` lengths from ``most`` down to half of it, the first the longest."""
    return [max(1, int(most * (1.0 - 0.5 * (i * GOLDEN % 1.0)))) if most else 0 for i in range(count)]


def _sequences(case):
    """(new tokens, tokens with them) of every sequence, in row order."""
    if case["kind"] == "append":
        count, rows = case["sequences"], case["rows"]
        each = _sizes(count, 1 << 20)
        new = [max(1, rows * e // sum(each)) for e in each]
        new[0] += rows - sum(new)
        while new[0] < 1:  # more sequences of one token than there were to share
            new[0] += 1
            new[new.index(max(new[1:]), 1)] -= 1
        return [(n, n + p) for n, p in zip(new, _sizes(count, case["prior"]))]
    decode = [(1, c) for c in _sizes(case["decode"], case["context"])]
    new, prior = _sizes(case["prompts"], case["chunk"]), _sizes(case["prompts"], case["prior"])
    return decode + [(n, n + p) for n, p in zip(new, prior)]


def _frequencies(rotary, scaling, factor=8.0, base=10000.0, original=4096):
    """fp64 radians a position of each pair, and the rotation's magnitude."""
    at = torch.arange(rotary // 2, dtype=torch.float64, device="cuda") * (2.0 / rotary)
    if scaling == "base":
        base = base * factor ** (rotary / (rotary - 2.0))
    f = torch.exp(-math.log(base) * at)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "bands":
        w = ((original * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return w * f + (1.0 - w) * f / factor, 0.1 * math.log(factor) + 1.0
    return f, 1.0


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _rotated(x, state):
    """[T, H, D] rotated by the rows' positions, in the type of ``x``."""
    f, magnitude = state["frequencies"], state["magnitude"]
    angle = state["positions"].double()[:, None] * f
    cos, sin = (g.to(x.dtype)[:, None, :] for g in (torch.cos(angle) * magnitude, torch.sin(angle) * magnitude))
    half, rotary = len(f), 2 * len(f)
    if state["interleaved"]:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    else:
        a, b = x[..., :half], x[..., half:rotary]
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(turned, -1).flatten(-2) if state["interleaved"] else torch.cat(turned, -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_rope(state):
    x = state["x"]
    return _rotated(x.float(), state).to(x.dtype)


def _stored(x, scale, dtype):
    """fp64 [T, H, D] as the cache's bytes or bf16 bits."""
    if dtype == torch.bfloat16:
        return x.to(dtype).view(torch.int16)
    return (x / scale.double()[:, None]).clamp(-448.0, 448.0).to(dtype).view(torch.uint8)


def _plain_append(state):
    positions, slots, table = state["positions"], state["row_slots"], state["table"]
    page_size = state["keys"].shape[2]
    live = (positions >= 0) & (slots >= 0)
    page = table[slots.clamp(min=0), positions.clamp(min=0) // page_size].long()
    live = torch.nonzero(live & (page >= 0)).squeeze(1)
    page, token = page[live], positions[live] % page_size
    k = _rotated(state["k"].double(), state)
    for rows, cache, scale in ((k, state["keys"], state["k_scale"]),
                               (state["v"].double(), state["values"], state["v_scale"])):
        bits = _stored(rows[live], scale, cache.dtype)
        cache.view(bits.dtype)[page, :, token] = bits
    q = _rotated(state["q"].float(), state).to(torch.bfloat16)
    return q, state["keys"], state["values"]


def _gathered(cache, scale, table, most):
    """Cached rows of every sequence: fp32 [n, kv heads, most, D], and which are mapped."""
    at = torch.arange(most, device=table.device)
    page = table[:, at // cache.shape[2]].long()
    bits = cache.view(torch.int16 if cache.dtype == torch.bfloat16 else torch.uint8)
    rows = bits[page.clamp(min=0), :, (at % cache.shape[2])[None, :]].view(cache.dtype)
    rows = rows.permute(0, 2, 1, 3).float()
    mapped = page >= 0
    return torch.where(mapped[:, None, :, None], rows * scale[:, None, None], 0.0), mapped


def _plain_attend(state):
    q, bounds, lengths = state["q"], state["boundaries"].long(), state["lengths"].long()
    rows_most, keys_most = state["rows_most"], state["keys_most"]
    total, heads, dim = q.shape
    kv_heads = state["keys"].shape[1]
    group, count = heads // kv_heads, len(lengths)
    new = bounds[1:] - bounds[:-1]
    j = torch.arange(rows_most, device=q.device)
    row = bounds[:-1, None] + j
    live = j < new[:, None]
    x = q.float()[row.clamp(max=total - 1)].reshape(count, rows_most, kv_heads, group, dim)
    x = x.permute(0, 2, 1, 3, 4).reshape(count, kv_heads, rows_most * group, dim) * state["scale"]
    table = state["table"][state["sequence_slots"]]
    keys, mapped = _gathered(state["keys"], state["k_scale"], table, keys_most)
    values, _ = _gathered(state["values"], state["v_scale"], table, keys_most)
    scores = torch.matmul(x, keys.transpose(2, 3).contiguous()).reshape(count, kv_heads, rows_most, group, keys_most)
    position = (lengths - new)[:, None] + j  # [n, rows]
    key = torch.arange(keys_most, device=q.device)
    seen = mapped[:, None, :] & (key <= position[..., None]) & live[..., None]
    if state["window"]:
        seen &= key > position[..., None] - state["window"]
    seen = seen[:, None, :, None, :]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    norm = scores.sum(-1)
    out = torch.matmul(scores.reshape(count, kv_heads, rows_most * group, keys_most), values)
    out = out.reshape(count, kv_heads, rows_most, group, dim) / torch.where(norm == 0, 1.0, norm)[..., None]
    out = out.permute(0, 2, 1, 3, 4).reshape(count, rows_most, heads, dim).to(torch.bfloat16)
    result = torch.zeros_like(q)
    result[row[live]] = out[live]
    return result


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _package():
    path = str(Path(__file__).resolve().parents[1] / "drama-3-single-b300-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from drama3_amd import attention

    return attention


def _own_rope(state):
    return state["package"].apply_rope(state["x"], state["positions"], state["rope"])


def _own_append(state):
    q = state["package"].append_paged(state["cache"], state["k"], state["v"], state["positions"], state["row_slots"],
                                      rope=state["rope"], q=state["q"])
    return q, state["keys"], state["values"]


def _own_attend(state):
    return state["package"].paged_attention(state["q"], state["cache"], state["layout"], state["lengths"],
                                            scale=state["scale"], window=state["window"] or None)


# ---------------------------------------------------------------------------
def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _cache_rows(gen, pages, kv_heads, page, dim, dtype):
    if dtype == torch.bfloat16:
        return _normal(gen, pages, kv_heads, page, dim)
    return (_normal(gen, pages, kv_heads, page, dim) * 40).clamp(-448, 448).to(dtype)


def _paged(case, gen, state, sequences):
    """A cache that holds the sequences, in pages of no order: some slots and table entries go unused."""
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    count = len(sequences)
    pages = [-(-total // page) for _, total in sequences]
    slots, wide = count + 3, max(pages) + 1
    order = torch.randperm(sum(pages) + 2, generator=gen, device="cuda")
    slot = torch.randperm(slots, generator=gen, device="cuda")[:count]
    owner = torch.repeat_interleave(torch.arange(count, device="cuda"), torch.tensor(pages, device="cuda"))
    first = torch.tensor([sum(pages[:i]) for i in range(count)], device="cuda")
    table = torch.full((slots, wide), -1, dtype=torch.int32, device="cuda")
    table[slot[owner], torch.arange(len(owner), device="cuda") - first[owner]] = order[: len(owner)].int()
    dtype = getattr(torch, case["cache"])
    state["keys"] = _cache_rows(gen, sum(pages) + 2, kv_heads, page, dim, dtype)
    state["values"] = _cache_rows(gen, sum(pages) + 2, kv_heads, page, dim, dtype)
    state["table"], state["sequence_slots"] = table, slot
    if dtype == torch.bfloat16:
        state["k_scale"] = state["v_scale"] = torch.ones(kv_heads, device="cuda")
        scales = {}
    else:  # what keys and values of a head are divided by before they are rounded
        state["k_scale"] = (1 + torch.rand(kv_heads, generator=gen, device="cuda")) / 64
        state["v_scale"] = (1 + torch.rand(kv_heads, generator=gen, device="cuda")) / 64
        scales = dict(k_scale=state["k_scale"], v_scale=state["v_scale"])
    if own:
        state["cache"] = _package().PagedCache(state["keys"], state["values"], table, **scales)


def _turning(case, state, rotary, scaling):
    state["frequencies"], state["magnitude"] = _frequencies(rotary, scaling)
    state["interleaved"] = case["interleaved"]
    if own:
        state["rope"] = _package().prepare_rope(rotary, interleaved=case["interleaved"], scaling=scaling,
                                                factor=8.0, original_length=4096)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"kind": kind}
    if own:
        state["package"] = _package()
    if kind == "rope":
        state["x"] = _normal(gen, case["rows"], case["heads"], case["dim"], dtype=getattr(torch, case["dtype"]))
        state["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=gen, device="cuda")
        _turning(case, state, case["rotary"], case["scaling"])
        return state
    sequences = _sequences(case)
    heads, kv_heads, dim, spare = case["heads"], case["kv_heads"], case["dim"], case["spare"]
    rows = sum(n for n, _ in sequences)
    _paged(case, gen, state, sequences)
    new = torch.tensor([n for n, _ in sequences], device="cuda")
    lengths = torch.tensor([t for _, t in sequences], dtype=torch.int32, device="cuda")
    bounds = torch.cat((new.new_zeros(1), new.cumsum(0)))
    if kind == "append":
        # One projection's result: queries, keys and values side by side.
        qkv = _normal(gen, rows + spare, heads + 2 * kv_heads, dim)
        state["q"], state["k"], state["v"] = qkv.split((heads, kv_heads, kv_heads), 1)
        owner = torch.repeat_interleave(torch.arange(len(sequences), device="cuda"), new)
        at = torch.arange(rows, device="cuda") - bounds[owner] + (lengths - new)[owner]
        state["positions"] = torch.cat((at, at.new_zeros(spare)))
        state["row_slots"] = torch.cat((state["sequence_slots"][owner], at.new_full((spare,), -1)))
        _turning(case, state, case["rotary"], "none")
        return state
    state["q"] = _normal(gen, rows + spare, heads, dim) * 1.5
    state["boundaries"], state["lengths"] = bounds.int(), lengths
    state["rows_most"], state["keys_most"] = max(n for n, _ in sequences), max(t for _, t in sequences)
    state["scale"], state["window"] = dim ** -0.5, case["window"]
    if own:
        from drama3_amd.packed_prefill import PackedLayout

        state["layout"] = PackedLayout(state["boundaries"], state["sequence_slots"], state["rows_most"])
    return state


def run(state):
    if own:
        return {"rope": _own_rope, "append": _own_append, "attend": _own_attend}[state["kind"]](state)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[state["kind"]](state)


def work(case):
    kind, dim = case["kind"], case["dim"]
    if kind == "rope":
        count = case["rows"] * case["heads"]
        size = 4 if case["dtype"] == "float32" else 2
        # read and written once; four products and two sums a pair
        return {"bytes": 2 * count * dim * size + 8 * case["rows"], "flops": 3 * count * case["rotary"]}
    heads, kv_heads = case["heads"], case["kv_heads"]
    size = 2 if case["cache"] == "bfloat16" else 1
    sequences = _sequences(case)
    rows = sum(n for n, _ in sequences)
    if kind == "append":
        every = rows + case["spare"]  # the queries of spare rows are rotated too
        return {"bytes": every * (4 * heads * dim + 16) + rows * 2 * kv_heads * dim * (2 + size),
                "flops": 3 * (every * heads + rows * kv_heads) * case["rotary"]}
    window = case["window"] or 1 << 40
    attended = keys = 0
    for new, total in sequences:
        first = total - new
        keys += min(total, window + new - 1)
        whole = max(0, min(total, window) - first)  # rows that see all keys up to their own
        attended += whole * first + whole * (whole + 1) // 2 + (new - whole) * min(window, total)
    return {"bytes": (2 * rows + case["spare"]) * heads * dim * 2 + 2 * keys * kv_heads * dim * size,
            "flops": 4 * attended * heads * dim}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope(x, positions, rotary, interleaved, scaling):
    """Every pair as a complex number, turned by a unit one."""
    s, original, base = 8.0, 4096.0, 10000.0
    magnitude = 1.0
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device=x.device)
    if scaling == "base":
        base *= s ** (rotary / (rotary - 2))
    f = base ** (-i / rotary)
    if scaling == "linear":
        f = f / s
    elif scaling == "bands":
        keep = torch.clamp((original * f / math.tau - 1) / 31, 0, 1)
        f = f * (keep + (1 - keep) / s)
        magnitude = 1 + math.log(s) / 10
    turn = torch.polar(torch.full((len(x), 1, rotary // 2), magnitude, dtype=torch.float64, device=x.device),
                       (positions.double()[:, None] * f)[:, None, :])
    pairs = x[..., :rotary].double()
    pairs = pairs.unflatten(-1, (-1, 2) if interleaved else (2, -1))
    pairs = pairs if interleaved else pairs.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = turned if interleaved else turned.transpose(-1, -2)
    out = x.double().clone()
    out[..., :rotary] = turned.flatten(-2)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(state["x"], state["positions"], case["rotary"], case["interleaved"], case["scaling"])
    page = case["page"]
    table = state["table"].tolist()
    slots = state["sequence_slots"].tolist()
    sequences = _sequences(case)
    if kind == "append":
        q, k = (_exact_rope(state[n], state["positions"], case["rotary"], case["interleaved"], "none") for n in "qk")
        kept = [state["keys"].double(), state["values"].double()]
        at = 0
        for (new, total), slot in zip(sequences, slots):
            for p in range((total - new) // page, -(-total // page)):  # the part of page p that the new tokens fill
                low, high = max(total - new, p * page), min(total, (p + 1) * page)
                rows = slice(at + low - (total - new), at + high - (total - new))
                for cache, fresh, scale in ((kept[0], k, state["k_scale"]), (kept[1], state["v"].double(), state["v_scale"])):
                    fresh = fresh[rows] / scale.double()[:, None]
                    if case["cache"] != "bfloat16":
                        fresh = fresh.clamp(-448, 448)
                    cache[table[slot][p], :, low - p * page: high - p * page] = fresh.transpose(0, 1)
            at += new
        return q, kept[0], kept[1]
    q = state["q"].double()
    out = torch.zeros_like(q)
    group, scale = case["heads"] // case["kv_heads"], state["scale"]
    at = 0
    for (new, total), slot in zip(sequences, slots):
        pages = table[slot][: -(-total // page)]
        low = max(0, total - new - case["window"] + 1) if case["window"] else 0
        key = torch.arange(low, total, device=q.device)
        own_position = torch.arange(total - new, total, device=q.device)[:, None]
        hidden = key > own_position
        if case["window"]:
            hidden = hidden | (key <= own_position - case["window"])
        for head in range(case["kv_heads"]):
            k, v = (state[n][pages, head].reshape(-1, case["dim"])[low:total].double() * state[s][head].double()
                    for n, s in (("keys", "k_scale"), ("values", "v_scale")))
            for member in range(group):
                mine = head * group + member
                scores = q[at: at + new, mine] @ k.T * scale
                scores[hidden] = -math.inf
                out[at: at + new, mine] = torch.softmax(scores, -1) @ v
        at += new
    return out
