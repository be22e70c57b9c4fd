"""Rotary positions, the paged cache and the attention over it in 64 bits, and
how the attention's kernels cut a call (numpy; test infrastructure)."""

from __future__ import annotations

import math

import numpy as np

BF16_HALF_STEP = 2.0 ** -8
F32_HALF_STEP = 2.0 ** -24
E4M3_MAX = 448.0


def rope(x, positions, frequencies, magnitude=1.0, interleaved=False):
    """x [T, H, D] (float64), radians a position [R / 2] -> rotated [T, H, D] and
    the sum |a| + |b| of each column's pair (0 where nothing turns)."""
    half = len(frequencies)
    # The angle's whole turns go before sine and cosine see it; long double keeps far positions exact.
    turns = np.longdouble(positions)[:, None] * (np.longdouble(frequencies) / (2 * np.longdouble(np.pi)))
    angle = ((turns - np.rint(turns)) * 2 * np.longdouble(np.pi)).astype(np.float64)[:, None, :]
    cos, sin = magnitude * np.cos(angle), magnitude * np.sin(angle)
    first = np.arange(half) * 2 if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    a, b = x[..., first], x[..., second]
    out, size = x.astype(np.float64).copy(), np.zeros(x.shape)
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = magnitude * (np.abs(a) + np.abs(b))
    return out, size


def rope_error(size):
    """What an fp32 rotation may be off by before its rounding, for pairs of that
    size: the remaining turn rounded to fp32 (at most 2^-25 turns), sine and
    cosine of it (two steps of 2^-23 near 1), their product with the magnitude,
    two products and a sum."""
    return size * (2 * math.pi * 2.0 ** -25 + 2 * 2.0 ** -23 + 4 * F32_HALF_STEP)


def e4m3(x):
    """The e4m3 values nearest to x, ties to the even code, magnitudes above 448 to 448."""
    x = np.clip(x, -E4M3_MAX, E4M3_MAX)
    exponent = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    step = np.exp2(exponent - 3)
    return np.rint(x / step) * step


def places(table, slots, positions, page_size, pages):
    """(page, token) of each row, page -1 where it goes nowhere."""
    out = []
    for slot, position in zip(slots, positions):
        page = -1
        if 0 <= slot < len(table) and 0 <= position < table.shape[1] * page_size:
            page = int(table[slot, position // page_size])
            page = page if 0 <= page < pages else -1
        out.append((page, int(position) % page_size))
    return out


def attention(q, keys, values, table, boundaries, slots, lengths, scale, window=None):
    """q [T, H, D], keys / values [pages, kv heads, P, D] (float64) -> (out, bound on
    what an fp32 evaluation with weights rounded to bf16 may be off by before
    its own rounding, rows that belong to a sequence)."""
    pages, kv_heads, page_size, dim = keys.shape
    group = q.shape[1] // kv_heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    owned = np.zeros(len(q), dtype=bool)
    for i, slot in enumerate(slots):
        first, end = (min(max(int(b), 0), len(q)) for b in boundaries[i:i + 2])
        owned[first:end] = True
        if not 0 <= slot < len(table):
            continue
        before = int(lengths[i]) - (end - first)
        for row in range(first, end):
            position = before + row - first
            at = np.arange(max(0, position - window + 1) if window else 0,
                           max(0, min(position + 1, table.shape[1] * page_size)))
            page = table[slot, at // page_size]
            at, page = at[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
            if len(at) == 0:
                continue
            for head in range(q.shape[1]):
                k, v = (t[page, head // group, at % page_size] for t in (keys, values))
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k @ q[row, head] * scale
                    w = np.exp(s - s.max())
                    out[row, head] = (w @ v) / w.sum()
                    # Relative error of a weight: the score's fp32 sum (its terms' sizes, the
                    # products by scale), the exponent's difference, 2^x itself; then of the sums
                    # over keys and the rescalings at growing maxima (at most one per 16 keys);
                    # each counted in numerator and denominator.  The weights' own rounding to bf16 may
                    # be in both: sum w (1 + d) v / sum w (1 + d) is off by sum w d (v - out) / sum w (1 + d).
                    sizes = (np.abs(k) @ np.abs(q[row, head])).max() * abs(scale)
                    rel = (dim + 8) * 2 * F32_HALF_STEP * sizes + 4 * F32_HALF_STEP * (s.max() - s.min()) + 2.0 ** -21
                    rel += (len(at) + 64) * 2 * F32_HALF_STEP + (len(at) // 16 + 8) * 2.0 ** -21
                    size = (w @ np.abs(v)) / w.sum() + np.abs(out[row, head])
                    bound[row, head] = size * (BF16_HALF_STEP / (1 - BF16_HALF_STEP) + 2 * rel * (1 + BF16_HALF_STEP))
    return out, bound, owned


# ---------------------------------------------------------------------------
# How a call is cut, as the kernels do it
# ---------------------------------------------------------------------------
BLOCK = 64
CUS = 256
ALONE, LEAST, LEAST_SPLIT = 512, 4, 4


def cut(rows, q_heads, kv_heads, boundaries, lengths, capacity, max_length, dim=128, window=0):
    """(units, bounds): every workgroup's (sequence, tile, single token or not, part
    or None, key range, the tile's range, packed rows), in the order of its keys,
    and the sizes that bound them."""
    group = q_heads // kv_heads
    all_single = max_length <= 1
    slices, count = -(-group // 16), len(lengths)
    some = min(count, rows)
    tile_rows = 256 if (dim == 128 and rows * q_heads >= 512 * 128 and max_length * group >= 4096
                        and some * kv_heads <= 1 << 22) else 128
    tile_tokens = 1 if all_single else tile_rows // group + 2
    single_tiles = (rows if all_single else some) * slices
    shift = 6
    while capacity <= ALONE and capacity > 1 << shift:
        shift += 1
    while (((capacity - 1) >> shift) + 1) * single_tiles >= 1 << 30:
        shift += 1
    most_blocks = ((capacity - 1) >> shift) + 1
    least = LEAST if most_blocks > 1 else 1
    a_cu = 1 if not all_single else (4 if dim == 64 else 2)
    shares = min(-(-single_tiles * most_blocks // least), max(1, a_cu * CUS // kv_heads)) if count else 0
    target = max(1, (1 if tile_rows == 256 else 2) * CUS // kv_heads)
    tiled = not all_single and count > 0
    tiles_most = rows * group // tile_rows + some if tiled else 0
    split_tiles = tiled and -(-capacity // BLOCK) > LEAST_SPLIT
    bounds = {"shares": shares, "tile_rows": tile_rows, "single_parts": 2 * shares if shares > 1 and most_blocks > 1 else 0,
              "tile_units": tiles_most + (target if split_tiles else 0), "tile_parts": 2 * target if split_tiles else 0,
              "split_tiles": min(tiles_most, target) if split_tiles else 0}
    most_tile_blocks, work_shift = -(-capacity // BLOCK), 0
    while tiles_most * (((most_tile_blocks - 1) >> work_shift) + 1) >= 1 << 31:
        work_shift += 1
    sequences, work, total = [], 0, 0
    for i in range(count):
        b0, b1 = (min(max(int(b), 0), rows) for b in boundaries[i:i + 2])
        tokens, length = max(b1 - b0, 0), max(int(lengths[i]), 0)
        single = all_single or tokens == 1
        tiles = tokens * slices if single else -(-tokens * group // tile_rows)
        size = shift if single else 6
        keys = min(length, capacity)
        if window:
            keys = min(keys, window + tile_tokens + (1 << size))
        blocks = max(1, -(-keys // (1 << size)))
        sequences.append((tokens, length, single, tiles, blocks))
        if single:
            total += tiles * blocks
        else:
            work += tiles * -(-blocks >> work_shift)
    assert work < 1 << 31
    inverse = min((1 << 32) // target + 1, (1 << 32) - 1)
    quotient = (work + target - (target > 1)) * inverse >> 32  # rounded up, or one more
    assert -(-work // target) <= quotient <= -(-work // target) + 1
    even = min(quotient, (1 << 30) >> work_shift) << work_shift
    chunk = max(even, (2 * LEAST_SPLIT if even > 1 else LEAST_SPLIT) if split_tiles else 1 << 30)
    each = max(least, -(-total // max(shares, 1)))
    units, part, at = [], 0, 0
    for i, (tokens, length, single, tiles, blocks) in enumerate(sequences):
        for tile in range(tiles):
            if single:
                low_token = high_token = tile // slices
                first = low_token * group + 16 * (tile % slices)
                packed = (first, min(first + 16, (low_token + 1) * group) - 1)
            else:
                packed = (tile * tile_rows, min((tile + 1) * tile_rows, tokens * group) - 1)
                low_token, high_token = packed[0] // group, packed[1] // group
            before = length - tokens
            size = shift if single else 6
            end = min(max(before + high_token + 1, 0), capacity)
            seen = before + low_token - window + 1 if window else 0
            start = min(max(seen, 0), end)
            aligned = start >> size << size

            def keys(low, high):
                return min(max(low, start), end), max(min(high, end), min(max(low, start), end))

            if single:
                w = at // each
                while w * each < at + blocks:
                    low, high = max(w * each, at) - at, min((w + 1) * each, at + blocks) - at
                    whole = high - low == blocks
                    units.append((i, tile, True, None if whole else 2 * w + (low == 0),
                                  keys(aligned + (low << size), aligned + (high << size)), (start, end), packed))
                    w += 1
                at += blocks
            else:
                splits = -(-blocks // chunk)
                step = -(-(-(-(end - aligned) // BLOCK)) // splits) * BLOCK
                for s in range(splits):
                    units.append((i, tile, False, None if splits == 1 else part + tile * splits + s,
                                  keys(aligned + s * step, aligned + (s + 1) * step), (start, end), packed))
        if not single and -(-blocks // chunk) > 1:
            part += tiles * -(-blocks // chunk)
    return units, bounds | {"each": each, "total": total}
