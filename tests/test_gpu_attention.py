"""Rotary positions, the paged append and the attention over the paged cache
against the 64-bit oracle, within the bounds that fp32 evaluation and one
rounding have (derived in the oracle), at the sizes, strides, masks and tables
where they can go wrong."""

import numpy as np
import pytest
import torch

from oracle import attention as oa

pytestmark = pytest.mark.gpu

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def within(got, want, bound):
    """Every element within its bound; NaN and infinities exactly where the oracle has them."""
    got = f64(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    excess = np.abs(got[fine] - want[fine]) - bound[fine]
    assert (excess <= 0).all(), f"{(excess > 0).sum()} of {excess.size} beyond, worst by {excess.max()}"


def randn(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape)).to(BF16)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, heads, dim, rotary", [
    (1, 1, 2, 2), (1, 16, 256, 64), (3, 5, 128, 128), (2, 7, 80, 20), (5, 3, 96, 18), (1029, 2, 16, 16), (67, 40, 128, 32),
    (2100, 3, 64, 64), (9, 1, 33, 6), (4, 2, 1024, 1024)])
def test_rope(device, rows, heads, dim, rotary, dtype, interleaved):
    from drama3_amd.attention import apply_rope, prepare_rope, rope_frequencies

    rng = np.random.default_rng(rows * 1000 + dim)
    x = torch.from_numpy(rng.standard_normal((rows, heads, dim))).to(dtype)
    positions = rng.integers(0, 131072, rows)
    out = apply_rope(x.to(device), torch.from_numpy(positions).to(device),
                     prepare_rope(rotary, interleaved=interleaved, device=device))
    want, size = oa.rope(f64(x), positions, rope_frequencies(rotary), interleaved=interleaved)
    err = oa.rope_error(size)
    step = oa.BF16_HALF_STEP if dtype == BF16 else oa.F32_HALF_STEP
    within(out, want, np.where(size == 0, 0.0, err + step * (np.abs(want) + err)))
    assert out.dtype == dtype


@pytest.mark.parametrize("scaling, more", [("linear", {}), ("base", {}), ("bands", dict(original_length=2048)),
                                           ("bands", dict(original_length=2048, magnitude=0.75))])
def test_rope_scalings_and_positions_of_any_kind(device, scaling, more):
    from drama3_amd.attention import apply_rope, prepare_rope, rope_frequencies

    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((6, 2, 64)))
    positions = np.array([0, -1, -70000, (1 << 31) - 1, 12345678, 1])
    magnitude = more.get("magnitude", 0.1 * np.log(16.0) + 1 if scaling == "bands" else 1.0)
    want, size = oa.rope(x.numpy(), positions, rope_frequencies(48, 500000.0, scaling, 16.0, more.get("original_length", 0)),
                         magnitude)
    rope = prepare_rope(48, 500000.0, scaling=scaling, factor=16.0, device=device, **more)
    # A position's turns are an fp64 product: off by 2^-53 of up to 2^31 turns, twice (the frequency's own rounding).
    err = oa.rope_error(size) + size * 2 * np.pi * 2.0 ** -21
    got = [apply_rope(x.float().to(device), torch.from_numpy(positions).to(dtype).to(device), rope)
           for dtype in (torch.int32, torch.int64)]
    x32 = f64(x.float())
    want32, _ = oa.rope(x32, positions, rope_frequencies(48, 500000.0, scaling, 16.0, more.get("original_length", 0)), magnitude)
    within(got[0], want32, np.where(size == 0, 0.0, err + oa.F32_HALF_STEP * (np.abs(want) + err)))
    assert torch.equal(got[0], got[1])


def test_rope_strides_in_place_and_empty(device):
    from drama3_amd.attention import apply_rope, prepare_rope

    rng = np.random.default_rng(6)
    rope = prepare_rope(32, device=device)
    x = randn(rng, 37, 9, 64).to(device)
    positions = torch.arange(37, device=device) * 11
    want = apply_rope(x, positions, rope)
    wide = torch.zeros(37, 700, dtype=BF16, device=device)
    view = wide[:, 51:51 + 9 * 65].as_strided((37, 9, 64), (700, 65, 1), wide.storage_offset() + 51)  # odd strides and start
    view.copy_(x)
    assert torch.equal(apply_rope(view, positions, rope), want)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside rows
    assert torch.equal(apply_rope(swapped, positions, rope), want)
    before = wide.clone()
    assert apply_rope(view, positions, rope, out=view) is view and torch.equal(view, want)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[:, 51:51 + 9 * 65].as_strided((37, 9, 64), (700, 65, 1), 51).fill_(False)
    assert torch.equal(wide[keep], before[keep])
    assert apply_rope(x[:0], positions[:0], rope).shape == (0, 9, 64)


def test_rope_of_nan_and_infinities_stays_in_its_pairs(device):
    from drama3_amd.attention import apply_rope, prepare_rope

    x = torch.ones(2, 3, 64, dtype=BF16)
    x[0, 1, 3], x[1, 2, 60] = float("nan"), float("inf")
    out = apply_rope(x.to(device), torch.tensor([3, 4], device=device), prepare_rope(32, device=device)).cpu()
    bad = ~torch.isfinite(out)
    assert bad.nonzero().tolist() == [[0, 1, 3], [0, 1, 19], [1, 2, 60]]


# ---------------------------------------------------------------------------
# The paged append
# ---------------------------------------------------------------------------
def cache_of(rng, device, pages, page_size, kv_heads, dim, table, dtype=BF16, order="heads", scales=True):
    """A PagedCache of random contents, and its keys and values as float64."""
    from drama3_amd.attention import PagedCache

    parts = []
    for _ in range(2):
        x = torch.from_numpy(rng.standard_normal((pages, kv_heads, page_size, dim)))
        x = (x * 30).clamp(-448, 448).float().to(E4M3) if dtype == E4M3 else x.to(BF16)
        if order == "tokens":  # [pages, page_size, kv_heads, dim] memory
            bits = x.view(torch.uint8) if dtype == E4M3 else x
            x = bits.transpose(1, 2).contiguous().to(device).transpose(1, 2)
            x = x.view(E4M3) if dtype == E4M3 else x
        parts.append(x.to(device))
    more = {}
    if dtype == E4M3 and scales:
        more = {n: torch.from_numpy(rng.uniform(0.01, 0.05, kv_heads)).float().to(device) for n in ("k_scale", "v_scale")}
    cache = PagedCache(*parts, torch.from_numpy(np.asarray(table, dtype=np.int32)).to(device), **more)
    scale = [f64(more[n])[:, None, None] if n in more else 1.0 for n in ("k_scale", "v_scale")]
    return cache, f64(parts[0]) * scale[0], f64(parts[1]) * scale[1]


@pytest.mark.parametrize("dtype, order", [(BF16, "heads"), (BF16, "tokens"), (E4M3, "heads"), (E4M3, "tokens")])
@pytest.mark.parametrize("rows, heads, kv_heads, dim, rotary, page_size, interleaved", [
    (1, 4, 1, 64, 64, 16, False), (5, 16, 2, 256, 64, 16, True), (70, 6, 3, 128, 128, 4, False), (33, 8, 8, 64, 20, 1, True),
    (40, 4, 2, 16, 16, 8, False), (1500, 2, 1, 64, 32, 64, False)])
def test_append(device, rows, heads, kv_heads, dim, rotary, page_size, interleaved, dtype, order):
    from drama3_amd.attention import append_paged, prepare_rope, rope_frequencies

    rng = np.random.default_rng(rows + dim)
    slots, wide = 5, -(-rows // page_size) + 2
    pages = slots * wide
    table = rng.permutation(pages).reshape(slots, wide)
    table[1, 0], table[2, wide - 1] = -1, pages  # unmapped both ways
    cache, keys, values = cache_of(rng, device, pages, page_size, kv_heads, dim, table, dtype, order)
    # Distinct tokens, some of them nowhere: bad slots, negative and far positions.
    token = rng.permutation(slots * wide * page_size)[:rows]
    row_slots, positions = token // (wide * page_size), token % (wide * page_size)
    for i, (s, p) in enumerate([(-1, 0), (slots, 3), (0, -1), (0, wide * page_size), (2, 1 << 40), (1 << 40, 0)]):
        if rows > 8 + i:
            row_slots[i], positions[i] = s, p
    qkv = randn(rng, rows, heads + 2 * kv_heads, dim)
    q, k, v = qkv.to(device).split((heads, kv_heads, kv_heads), 1)
    before = [t.view(torch.uint8).clone() for t in (cache.keys, cache.values)] if order == "heads" else None
    out = append_paged(cache, k, v, torch.from_numpy(positions).to(device), torch.from_numpy(row_slots).to(device),
                       prepare_rope(rotary, interleaved=interleaved, device=device), q=q)
    f = rope_frequencies(rotary)
    safe = np.clip(positions, -1, 1 << 30)  # (turned wherever they go; the oracle's long double as well)
    want, size = oa.rope(f64(qkv), positions, f, interleaved=interleaved)
    err = oa.rope_error(size) + size * 2 * np.pi * np.abs(positions)[:, None, None] * 2.0 ** -52
    assert (safe == positions).sum() >= rows - 2
    within(out, want[:, :heads], np.where(size == 0, 0.0, err + oa.BF16_HALF_STEP * (np.abs(want) + err))[:, :heads])
    at = oa.places(table, row_slots, positions, page_size, pages)
    moved = np.zeros((pages, page_size), dtype=bool)
    scales = [f64(t)[:, None] if t is not None else 1.0 for t in (cache.k_scale, cache.v_scale)]
    for r, (page, t) in enumerate(at):
        if page < 0:
            continue
        moved[page, t] = True
        for store, part, scale, e in ((cache.keys, want[r, heads:heads + kv_heads], scales[0], err[r, heads:heads + kv_heads]),
                                      (cache.values, f64(qkv[r, heads + kv_heads:]), scales[1], 0.0)):
            got = f64(store[page, :, t].float())
            if dtype == BF16:
                within(torch.from_numpy(got), part, np.where(e == 0, 0, e + oa.BF16_HALF_STEP * (np.abs(part) + e)))
            else:  # a code nearest to a value within the rotation's error (and the division's)
                x = part / scale
                e = (e / scale + np.abs(x) * oa.F32_HALF_STEP)
                assert ((oa.e4m3(x - e) <= got) & (got <= oa.e4m3(x + e))).all()
    if before is not None:
        for store, old in ((cache.keys, before[0]), (cache.values, before[1])):
            same = (store.view(torch.uint8) == old).view(pages, kv_heads, page_size, -1).all(-1).all(1).cpu().numpy()
            assert same[~moved].all()


def test_append_without_rotation_or_queries(device):
    from drama3_amd.attention import append_paged

    rng = np.random.default_rng(8)
    cache, _, _ = cache_of(rng, device, 4, 16, 2, 128, [[2, 0], [1, 3]])
    k, v = randn(rng, 3, 2, 128).to(device), randn(rng, 3, 2, 128).to(device)
    positions, slots = torch.tensor([17, 0, 31], dtype=torch.int32, device=device), torch.tensor([0, 1, 1], device=device)
    assert append_paged(cache, k, v, positions, slots) is None
    assert torch.equal(cache.keys[0, :, 1], k[0]) and torch.equal(cache.values[0, :, 1], v[0])
    assert torch.equal(cache.keys[1, :, 0], k[1]) and torch.equal(cache.values[3, :, 15], v[2])
    q = randn(rng, 3, 4, 128).to(device)
    assert torch.equal(append_paged(cache, k, v, positions, slots, q=q), q)
    assert append_paged(cache, k[:0], v[:0], positions[:0], slots[:0]) is None


def test_append_e4m3_of_nan_and_large_values(device):
    from drama3_amd.attention import append_paged

    cache, _, _ = cache_of(np.random.default_rng(9), device, 1, 16, 1, 64, [[0]], E4M3, scales=False)
    v = torch.zeros(1, 1, 64, dtype=BF16, device=device)
    v[0, 0, :6] = torch.tensor([float("nan"), float("inf"), -float("inf"), 500.0, -449.0, 2.0 ** -10])
    append_paged(cache, v, v, torch.zeros(1, dtype=torch.int64, device=device), torch.zeros(1, dtype=torch.int64, device=device))
    for store in (cache.keys, cache.values):
        got = store[0, 0, 0, :6].float().cpu().tolist()
        assert got[0] != got[0] and got[1:] == [448.0, -448.0, 448.0, -448.0, 0.0]  # (half a step goes to the even code)


# ---------------------------------------------------------------------------
# The attention
# ---------------------------------------------------------------------------
def tables_for(rng, lengths, page_size, spare=2):
    """A page table for sequences in random slots: (table, slots, pages)."""
    need = [-(-max(int(n), 1) // page_size) for n in lengths]
    slots = rng.permutation(len(need) + 2)[:len(need)]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(need) + 2, max(need) + 1), -1)
    at = 0
    for slot, n in zip(slots, need):
        table[slot, :n] = order[at:at + n]
        at += n
    return table, slots, sum(need) + spare


def layout_of(device, boundaries, slots, max_length):
    from drama3_amd.packed_prefill import PackedLayout

    return PackedLayout(torch.tensor(np.asarray(boundaries), dtype=torch.int32, device=device),
                        torch.tensor(np.asarray(slots), dtype=torch.int64, device=device), max_length)


def check(out, q, keys, values, table, boundaries, slots, lengths, scale, window=None):
    want, bound, owned = oa.attention(f64(q), keys, values, table, boundaries, slots, lengths, scale, window)
    within(out, want, bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))
    got = f64(out)
    fine = np.isfinite(want) & (bound > 0)
    if fine.sum() > 4096:
        # Two independent roundings of at most half a step (weights, result): rms below 2^-8 sqrt(2/3) of the
        # values' own or, where values cancel, of the weights' share; 2^-8 of the mean size bounds both.
        rms = np.sqrt(np.mean((got - want)[fine] ** 2))
        assert rms <= oa.BF16_HALF_STEP * np.sqrt(np.mean((bound[fine] / oa.BF16_HALF_STEP) ** 2))
    return owned


CASES = {  # new tokens, cached ones with them
    "one": ([1], [1]), "one_key_short_of_a_block": ([1, 1, 1], [63, 64, 65]), "empty": ([1, 0, 1, 1], [5, 3, 0, 70]),
    "decode": ([1] * 9, [1, 2, 31, 32, 33, 127, 128, 129, 500]), "long": ([1, 1], [4097, 300]),
    "pair": ([2, 1, 3], [2, 40, 90]), "prompts": ([33, 1, 70, 5], [33, 200, 70, 64]), "chunk": ([130], [517]),
    "short_table": ([4, 2], [2, 1]), "tail": ([17, 129], [2049, 129])}


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 1, 64), (6, 2, 128), (4, 4, 128), (4, 2, 256), (40, 2, 64), (17, 1, 128)])
@pytest.mark.parametrize("case", CASES)
def test_attention(device, case, heads, kv_heads, dim, dtype):
    from drama3_amd.attention import paged_attention

    new, lengths = CASES[case]
    rng = np.random.default_rng(sum(lengths) + heads + dim)
    page_size = int(rng.choice([1, 8, 16, 64, 256]))
    table, slots, pages = tables_for(rng, lengths, page_size)
    cache, keys, values = cache_of(rng, device, pages, page_size, kv_heads, dim, table, dtype,
                                   "tokens" if heads == 6 else "heads")
    first, behind = int(rng.integers(0, 2)), int(rng.integers(0, 3))
    boundaries = np.concatenate([[0], np.cumsum(new)]) + first
    q = (1.5 * randn(rng, boundaries[-1] + behind, heads, dim)).to(BF16)
    longest = max(new)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, longest),
                          torch.tensor(lengths, device=device))
    owned = check(out, q, keys, values, table, boundaries, slots, lengths, dim ** -0.5)
    assert not out[torch.from_numpy(~owned).to(device)].any()
    # The same bits from the same call, into given rows too; rows of no sequence stay.
    given = torch.full_like(out, 7.0)
    paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, longest),
                    torch.tensor(lengths, dtype=torch.int32, device=device), out=given)
    mine = torch.from_numpy(owned).to(device)
    assert torch.equal(given[mine], out[mine]) and (given[~mine] == 7.0).all()


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 1 << 40])
@pytest.mark.parametrize("new, lengths", [([1, 1, 1], [1, 300, 64]), ([150, 3, 1], [150, 333, 40])])
def test_window(device, window, new, lengths):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(window % 1000 + len(lengths) + lengths[0])
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, 64, table)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1], 6, 64)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)),
                          torch.tensor(lengths, device=device), scale=0.3, window=window)
    check(out, q, keys, values, table, boundaries, slots, lengths, 0.3, min(window, 1 << 20))


@pytest.mark.parametrize("new, lengths", [([1] * 6, [300, 40, 5, 100, 64, 9]), ([70, 5, 1, 1, 1, 1], [300, 40, 5, 100, 64, 9])])
def test_unmapped_pages_bad_slots_and_lengths(device, new, lengths):
    """Table entries outside the pages, slots outside the table, lengths below the
    new tokens', negative and past the table, boundaries past the rows."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(len(new) + new[0])
    table, slots, pages = tables_for(rng, lengths, 16)
    table[slots[0], 3], table[slots[0], 5], table[slots[3], :7] = -1, pages, -7
    table[slots[4], 0] = (1 << 31) - 1
    slots[1], slots[2] = -1, len(table)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, 128, table)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    boundaries[-1] += 5
    told = list(lengths)
    told[4], told[5] = (1 << 35), -3
    q = randn(rng, int(np.sum(new)), 4, 128)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)), torch.tensor(told, device=device))
    told[4] = (1 << 31) - 1  # what such a length reads as: every mapped token
    check(out, q, keys, values, table, boundaries, slots, told, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_attended_is_not_felt(device, dim, dtype, bad):
    """NaN and infinities in keys and values behind a length, before a window, in
    unmapped pages and in tokens newer than a row; where a row does attend them it
    has them."""
    from drama3_amd.attention import paged_attention

    if dtype == E4M3 and bad != bad:
        pass
    elif dtype == E4M3:
        pytest.skip("e4m3 has no infinities")
    rng = np.random.default_rng(dim)
    new, lengths = [40, 1, 1], [100, 77, 130]
    table, slots, pages = tables_for(rng, lengths, 16, spare=3)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, dim, table, dtype, scales=False)
    spoiled = [(table[slots[0], 6], 2), (table[slots[0], 6], 4), (table[slots[0], 6], 9), (table[slots[1], 4], 15),
               (table[slots[2], 0], 0)]  # positions 98, (behind the length) 100, 105; behind 77; before the window
    free = [p for p in range(pages) if p not in table]
    for page, token in spoiled + [(p, t) for p in free for t in range(16)]:
        column = int(rng.integers(0, dim))
        for store, plain in ((cache.keys, keys), (cache.values, values)):
            bits = store.view(torch.uint8) if dtype == E4M3 else store
            if dtype == E4M3:
                bits[page, 1, token, column] = 0x7f
            else:
                bits[page, 1, token, column] = bad
            plain[page, 1, token, column] = bad
    # Keys of the one that rows do attend stay finite: values alone, so that infinities come through as themselves.
    page, token = spoiled[0]
    clean = torch.from_numpy(rng.standard_normal(dim)).float().to(dtype)
    (cache.keys.view(torch.uint8) if dtype == E4M3 else cache.keys)[page, 1, token] = (
        clean.view(torch.uint8) if dtype == E4M3 else clean).to(device)
    keys[page, 1, token] = f64(clean.float())
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1], 4, dim)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, 40), torch.tensor(lengths, device=device),
                          window=90)
    want, bound, _ = oa.attention(f64(q), keys, values, table, boundaries, slots, lengths, dim ** -0.5, 90)
    rows = np.nonzero(~np.isfinite(want).all((1, 2)))[0].tolist()
    assert rows == [38, 39]  # the newest of the chunk that attend position 98
    within(out, want, bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))
    # Single tokens alone, by their own kernel.
    out = paged_attention(q[40:].to(device), cache, layout_of(device, [0, 1, 2], slots[1:], 1),
                          torch.tensor(lengths[1:], device=device), window=90)
    within(out, want[40:], (bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))[40:])


def test_large_scores(device):
    """Scores of many hundreds, rising along the keys (every block rescales) and falling."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(12)
    lengths = [400, 400]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 1, 64, table)
    for slot, ramp in zip(slots, (np.linspace(-8, 8, 400), np.linspace(8, -8, 400))):
        for t in range(400):
            row = torch.full((64,), float(ramp[t])).to(BF16)
            cache.keys[table[slot, t // 16], 0, t % 16] = row.to(device)
            keys[table[slot, t // 16], 0, t % 16] = f64(row)
    for new in ([1, 1], [9, 30]):
        boundaries = np.concatenate([[0], np.cumsum(new)])
        q = torch.ones(boundaries[-1], 3, 64, dtype=BF16) * torch.tensor([1.0, -1.0, 0.25]).to(BF16)[:, None]
        out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)),
                              torch.tensor(lengths, device=device), scale=1.0)
        check(out, q, keys, values, table, boundaries, slots, lengths, 1.0)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("step", [0.5, 7.0, 7.9, 8.1, 40.0, -7.9])
def test_scores_that_climb_block_by_block(device, dim, step):
    """Scores `step` powers of two higher every 32 keys, up and down in turns of five, with
    values of up to 2^90: under the rise of a row's base, at it and above it."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(31)
    lengths = [700, 333]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 1, dim, table)
    for store, mine in ((cache.keys, keys), (cache.values, values)):
        rows = torch.from_numpy(mine).to(BF16)
        if mine is values:
            rows *= 2.0 ** 90
        else:
            rows[...] = 0
            for slot, length in zip(slots, lengths):
                for t in range(length):
                    block = t // 32
                    # (the sum of dim equal products is the score)
                    rows[table[slot, t // 16], 0, t % 16] = step * (5 - abs(block % 10 - 5)) / dim
        store.copy_(rows.to(device))
        mine[...] = f64(rows)
    for new in ([1, 1], [140, 30]):
        boundaries = np.concatenate([[0], np.cumsum(new)])
        q = torch.ones(boundaries[-1], 2, dim, dtype=BF16) * torch.tensor([1.0, 0.5]).to(BF16)[:, None]
        out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)),
                              torch.tensor(lengths, device=device), scale=float(np.log(2)))
        check(out, q, keys, values, table, boundaries, slots, lengths, float(np.log(2)))


def test_graphs_replayed_at_once(device):
    """Two captured calls, each with parts of its own, replayed on two streams at the same time."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(32)
    lengths = [5000, 3000, 64]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, _, _ = cache_of(rng, device, pages, 16, 2, 128, table)
    told = torch.tensor(lengths, device=device)
    calls, wants, graphs = [], [], []
    for new in ([1, 1, 1], [40, 1, 20]):
        layout = layout_of(device, np.concatenate([[0], np.cumsum(new)]), slots, max(new))
        q = randn(rng, sum(new), 16, 128).to(device)
        wants.append(paged_attention(q, cache, layout, told))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention(q, cache, layout, told)
        calls.append((q, layout, out)), graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for _, _, out in calls:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for (_, _, out), want in zip(calls, wants))


@pytest.mark.parametrize("hint", [0, 1, 2, 100000])
def test_longest_sequence_only_chooses_the_kernels(device, hint):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(13)
    new, lengths = [1, 20, 0, 3], [500, 300, 4, 3]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, 128, table)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1], 36, 128)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, hint), torch.tensor(lengths, device=device))
    check(out, q, keys, values, table, boundaries, slots, lengths, 128 ** -0.5)


def test_many_sequences_and_strided_rows(device):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(14)
    new = rng.integers(0, 3, 150)
    lengths = new + rng.integers(0, 90, 150)
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 1, 64, table)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    rows = int(boundaries[-1])
    wide = randn(rng, rows, 3 * 77).to(device)
    q = wide.as_strided((rows, 3, 64), (231, 77, 1), 5)
    out = torch.zeros(rows, 4, 80, dtype=BF16, device=device)
    for hint in (1, 2):
        paged_attention(q, cache, layout_of(device, boundaries, slots, hint), torch.tensor(lengths, device=device),
                        out=out[:, 1:, 8:72])
        check(out[:, 1:, 8:72], q, keys, values, table, boundaries, slots, lengths, 0.125)
        assert not out[:, 0].any() and not out[..., :8].any() and not out[..., 72:].any()


def test_no_rows_and_no_sequences(device):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(15)
    cache, _, _ = cache_of(rng, device, 2, 16, 1, 64, [[0, 1]])
    none = torch.zeros(0, dtype=torch.int64, device=device)
    q = randn(rng, 3, 2, 64).to(device)
    assert paged_attention(q[:0], cache, layout_of(device, [0], [], 1), none).shape == (0, 2, 64)
    for hint in (1, 5):
        assert not paged_attention(q, cache, layout_of(device, [0], [], hint), none).any()
        given = torch.ones_like(q)
        assert (paged_attention(q, cache, layout_of(device, [0], [], hint), none, out=given) == 1).all()
        assert not paged_attention(q, cache, layout_of(device, [0, 0], [0], hint), torch.tensor([5], device=device)).any()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_pages_past_32_bit_offsets(device, dtype):
    """A cache of more than 2^32 elements, of which a few far pages are used."""
    from drama3_amd.attention import PagedCache, append_paged, paged_attention

    rng = np.random.default_rng(16)
    pages = (1 << 32) // (4 * 64 * 128) + 40
    keys = torch.empty(pages, 4, 64, 128, dtype=dtype, device=device)
    values = torch.empty_like(keys)
    table = np.array([[pages - 1, pages - 3, 2, pages - 20]])
    cache = PagedCache(keys, values, torch.tensor(table, dtype=torch.int32, device=device))
    k, v, q = randn(rng, 200, 4, 128), randn(rng, 200, 4, 128), randn(rng, 200, 8, 128)
    append_paged(cache, k.to(device), v.to(device), torch.arange(200, device=device), torch.zeros(200, dtype=torch.int64, device=device))
    small_k = np.stack([f64(keys[p].float()) for p in table[0]])
    small_v = np.stack([f64(values[p].float()) for p in table[0]])
    for new in (1, 200):
        out = paged_attention(q[-new:].to(device), cache, layout_of(device, [0, new], [0], new), torch.tensor([200], device=device))
        # (the last, unused part of the fourth page is uninitialised memory)
        check(out, q[-new:], small_k, small_v, np.array([[0, 1, 2, 3]]), [0, new], [0], [200], 128 ** -0.5)


# ---------------------------------------------------------------------------
# Many rows: tiles of two groups of waves, results larger than the L2s
# ---------------------------------------------------------------------------
def reference(q, keys, values, table, boundaries, slots, lengths, scale, window=None):
    """The oracle's ``attention`` in torch float64 on the device, whole sequences at a time
    (q, keys, values there; table and the rest as in the oracle): (out, bound)."""
    pages, kv_heads, page_size, dim = keys.shape
    group = q.shape[1] // kv_heads
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for first, end, slot, length in zip(boundaries, boundaries[1:], slots, lengths):
        if first == end:
            continue
        at = np.arange(min(int(length), table.shape[1] * page_size))
        page = table[slot, at // page_size]
        kept = (page >= 0) & (page < pages)
        at, page = (torch.from_numpy(x[kept]).to(q.device) for x in (at, page))
        position = torch.arange(int(length) - int(end - first), int(length), device=q.device)[:, None]
        hidden = at > position
        if window:
            hidden |= at <= position - window
        none = hidden.all(1)
        count = len(at)
        for head in range(q.shape[1]):
            k, v = (t[page.long(), head // group, at % page_size] for t in (keys, values))
            mine = q[first:end, head]
            s = (mine @ k.T * scale).masked_fill(hidden, -torch.inf)
            low, top = s.masked_fill(hidden, torch.inf).amin(1), s.amax(1)
            w = torch.exp(s - top.masked_fill(none, 0)[:, None])
            total = w.sum(1).masked_fill(none, 1)[:, None]
            # (a value that a row does not attend takes no part, whatever it is)
            bad = ~torch.isfinite(v)
            clean = v.masked_fill(bad, 0)
            o = w @ clean / total
            if bad.any():
                for t in bad.any(1).nonzero().squeeze(1).tolist():
                    o[~hidden[:, t]] += torch.where(bad[t], v[t], 0.0)
            sizes = (mine.abs() @ k.abs().T).masked_fill(hidden, 0).nan_to_num(0).amax(1) * abs(scale)
            rel = (dim + 8) * 2 * oa.F32_HALF_STEP * sizes + 4 * oa.F32_HALF_STEP * (top - low) + 2.0 ** -21
            rel = (rel + (count + 64) * 2 * oa.F32_HALF_STEP + (count // 16 + 8) * 2.0 ** -21).masked_fill(none, 0)[:, None]
            share = oa.BF16_HALF_STEP / (1 - oa.BF16_HALF_STEP) + 2 * rel * (1 + oa.BF16_HALF_STEP)
            out[first:end, head] = o.masked_fill(none[:, None], 0)
            bound[first:end, head] = (w @ clean.abs() / total + o.abs().nan_to_num(0, 0, 0)) * share
    return out, bound


def test_the_device_reference_is_the_oracle(device):
    rng = np.random.default_rng(20)
    new, lengths = [20, 1, 0, 9], [60, 33, 5, 4]
    table, slots, pages = tables_for(rng, lengths, 8)
    table[slots[0], 2] = -1
    _, keys, values = cache_of(rng, device, pages, 8, 2, 64, table)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1], 4, 64)
    values[table[slots[0], 6], 1, 5, 7] = np.inf
    want, bound, _ = oa.attention(f64(q), keys, values, table, boundaries, slots, lengths, 0.2, 25)
    got, sizes = reference(q.double().to(device), *(torch.from_numpy(t).to(device) for t in (keys, values)), table, boundaries,
                           slots, lengths, 0.2, 25)
    within(got, want, 1e-12 * (1 + np.abs(np.nan_to_num(want, posinf=0))))
    fine = np.isfinite(want)
    assert np.allclose(f64(sizes)[fine], bound[fine], rtol=0.01)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("new, lengths, window, page_size", [
    ([2100], [2400], None, 16), ([2049, 1, 33, 1, 0, 7], [2049, 900, 40, 3, 5, 700], None, 64),
    ([2300, 1], [2500, 600], 300, 1), ([2150], [2150], 64, 128)])
def test_many_rows(device, new, lengths, window, page_size, dtype):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(sum(new) + page_size)
    table, slots, pages = tables_for(rng, lengths, page_size)
    table[slots[0], len(table[0]) // 3] = -1
    cache, keys, values = cache_of(rng, device, pages, page_size, 8, 128, table, dtype)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1] + 3, 32, 128)
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)),
                          torch.tensor(lengths, device=device), window=window)
    want, bound = reference(q.double().to(device), *(torch.from_numpy(t).to(device) for t in (keys, values)), table, boundaries,
                            slots, lengths, 128 ** -0.5, window)
    want, bound = f64(want), f64(bound)
    within(out, want, bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows, heads, kv_heads, dim, window", [
    (2100, 32, 8, 128, None), (600, 4, 2, 128, 150), (700, 4, 2, 64, None), (300, 8, 8, 64, 100), (300, 4, 2, 256, None)])
def test_many_rows_do_not_feel_newer_values(device, rows, heads, kv_heads, dim, window, bad):
    """An infinity or a NaN among the values: in a block that some rows of a tile attend,
    others in part and others not at all, each row as if it were alone."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(21 + rows)
    lengths = [rows + 200]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, kv_heads, dim, table)
    for position in (rows + 199, rows - 3, rows - 2, rows // 2, 250, 201, 200, 199):
        page, token, head = table[slots[0], position // 16], position % 16, int(rng.integers(0, kv_heads))
        column = int(rng.integers(0, dim))
        cache.values[page, head, token, column] = bad
        values[page, head, token, column] = bad
    q = randn(rng, rows, heads, dim)
    out = paged_attention(q.to(device), cache, layout_of(device, [0, rows], slots, rows), torch.tensor(lengths, device=device),
                          window=window)
    want, bound = reference(q.double().to(device), *(torch.from_numpy(t).to(device) for t in (keys, values)), table, [0, rows],
                            slots, lengths, dim ** -0.5, window)
    assert (~torch.isfinite(want)).any(2).any(1).sum() > 50 and torch.isfinite(want).any(2).any(1).all()
    want, bound = f64(want), f64(bound)
    within(out, want, bound + oa.BF16_HALF_STEP * (np.abs(np.nan_to_num(want, nan=0, posinf=0, neginf=0)) + bound))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_past_the_caches(device, interleaved):
    """Results of more than 32 MB: rope and append, against fp64 on the device."""
    from drama3_amd.attention import PagedCache, append_paged, apply_rope, prepare_rope, rope_frequencies

    rng = np.random.default_rng(22)
    rows, heads, kv_heads, dim = 8300, 16, 2, 128
    qkv = randn(rng, rows, heads + 2 * kv_heads, dim).to(device)
    positions = torch.from_numpy(rng.permutation(rows)).to(device)
    rope = prepare_rope(dim, interleaved=interleaved, device=device)
    angle = positions.double()[:, None] * torch.tensor(rope_frequencies(dim), dtype=torch.float64, device=device)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    x = qkv.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :64], x[..., 64:])
    want = (a * cos - b * sin, a * sin + b * cos)
    want = torch.stack(want, -1).flatten(-2) if interleaved else torch.cat(want, -1)
    size = a.abs() + b.abs()
    size = size.repeat_interleave(2, -1) if interleaved else torch.cat((size, size), -1)
    err = oa.rope_error(size) + size * 1e-9  # (the angle's own 64 bits at 8300 positions)
    allowed = err + oa.BF16_HALF_STEP * (want.abs() + err)
    assert ((apply_rope(qkv, positions, rope).double() - want).abs() <= allowed).all()
    cache = PagedCache.empty(520, 16, kv_heads, dim, 2, 520, device=device)
    order = torch.randperm(520, device=device)
    cache.page_table[1] = order.int()
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    out = append_paged(cache, k, v, positions, torch.ones_like(positions), rope=rope, q=q)
    assert ((out.double() - want[:, :heads]).abs() <= allowed[:, :heads]).all()
    at = order[positions // 16], positions % 16
    assert ((cache.keys[at[0], :, at[1]].double() - want[:, heads:heads + kv_heads]).abs() <= allowed[:, heads:heads + kv_heads]).all()
    assert torch.equal(cache.values[at[0], :, at[1]], v)


@pytest.mark.parametrize("scale, k_sign", [(-0.1, 1.0), (0.0, 1.0), (0.1, -1.0)])
def test_scales_of_any_sign(device, scale, k_sign):
    from drama3_amd.attention import PagedCache, paged_attention

    rng = np.random.default_rng(23)
    new, lengths = [1, 40], [90, 70]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, 64, table, E4M3)
    cache = PagedCache(cache.keys, cache.values, cache.page_table, cache.k_scale * k_sign, cache.v_scale * -1)
    q = randn(rng, 41, 4, 64)
    for hint in (1, 40):
        out = paged_attention(q.to(device), cache, layout_of(device, [0, 1, 41], slots, hint), torch.tensor(lengths, device=device),
                              scale=scale)
        check(out, q, keys * k_sign, -values, table, [0, 1, 41], slots, lengths, scale)


# ---------------------------------------------------------------------------
# Used together
# ---------------------------------------------------------------------------
def test_prefill_then_decode_equals_attention_of_the_whole(device):
    """Prompts in two chunks, then single tokens, through append and attention with
    packed row metadata: every row as attention over the rotated rows at once."""
    from drama3_amd.attention import PagedCache, append_paged, paged_attention, prepare_rope, rope_frequencies
    from drama3_amd.packed_prefill import packed_row_metadata

    rng = np.random.default_rng(17)
    heads, kv_heads, dim, rotary = 8, 2, 64, 32
    total = [90, 41]
    qkv = [randn(rng, n, heads + 2 * kv_heads, dim) for n in total]
    cache = PagedCache.empty(20, 16, kv_heads, dim, 4, 8, device=device)
    order = rng.permutation(20)[:9]
    cache.page_table[3, :6] = torch.tensor(order[:6], dtype=torch.int32)
    cache.page_table[1, :3] = torch.tensor(order[6:], dtype=torch.int32)
    rope = prepare_rope(rotary, device=device)
    got = [[], []]
    for new in ([50, 7], [37, 31], [1, 1], [1, 1], [1, 1]):
        done = [sum(len(x) for x in g) for g in got]
        layout = layout_of(device, np.concatenate([[0], np.cumsum(new)]), [3, 1], max(new))
        rows = torch.cat([x[d:d + n] for x, d, n in zip(qkv, done, new)]).to(device)
        positions = torch.empty(len(rows), dtype=torch.int64, device=device)
        row_slots = torch.empty_like(positions)
        packed_row_metadata(layout.boundaries, layout.sequence_slots, len(rows), positions, row_slots)
        positions += torch.tensor(done, device=device).repeat_interleave(torch.tensor(new, device=device))
        q, k, v = rows.split((heads, kv_heads, kv_heads), 1)
        q = append_paged(cache, k, v, positions, row_slots, rope=rope, q=q)
        lengths = torch.tensor([d + n for d, n in zip(done, new)], device=device)
        out = paged_attention(q, cache, layout, lengths)
        for g, part in zip(got, out.split(new)):
            g.append(part)
    for x, g in zip(qkv, got):
        turned, size = oa.rope(f64(x[:, :heads + kv_heads]), np.arange(len(x)), rope_frequencies(rotary))
        # The operators round the rotated rows to bf16: so does the expectation, and a score may differ by a
        # step of both (where fp32 and 64 bits fall on two sides of a border).
        rounded = f64(torch.from_numpy(turned).float().to(BF16))
        keys = np.zeros((1, kv_heads, 128, dim))
        values = np.zeros((1, kv_heads, 128, dim))
        keys[0, :, :len(x)] = rounded[:, heads:].transpose(1, 0, 2)
        values[0, :, :len(x)] = f64(x[:, heads + kv_heads:]).transpose(1, 0, 2)
        want, bound, _ = oa.attention(rounded[:, :heads], keys, values, np.array([[0]]), [0, len(x)], [0], [len(x)], dim ** -0.5)
        flips = 2 * oa.BF16_HALF_STEP * 2 * 64 ** -0.5 * 16  # of a score of sizes up to 4 x 4, one element of each side
        bound = bound + 2 * flips * np.abs(values).max()
        within(torch.cat(g), want, bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))


def step_of(cache, layout, lengths, positions, slots, rows, heads, kv_heads, rope):
    from drama3_amd.attention import append_paged, paged_attention

    q, k, v = rows.split((heads, kv_heads, kv_heads), 1)
    q = append_paged(cache, k, v, positions, slots, rope=rope, q=q)
    return paged_attention(q, cache, layout, lengths)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 9]])
def test_captured_steps_replay_with_new_lengths_tables_and_rows(device, new):
    """Two captured steps of one cache, replayed in turn with eager work between,
    their inputs rewritten: every replay as the eager call."""
    from drama3_amd.attention import prepare_rope

    rng = np.random.default_rng(18 + new[0])
    heads, kv_heads, dim = 8, 2, 128
    table, slots, pages = tables_for(rng, [900, 700, 400], 16)
    cache, _, _ = cache_of(rng, device, pages, 16, kv_heads, dim, table)
    rope = prepare_rope(dim, device=device)
    rows = sum(new)
    steps = []
    for _ in range(2):
        layout = layout_of(device, np.concatenate([[0], np.cumsum(new)]), slots, max(new))
        state = dict(layout=layout, lengths=torch.tensor(new, device=device), rows=randn(rng, rows, heads + 2 * kv_heads, dim).to(device),
                     positions=torch.zeros(rows, dtype=torch.int64, device=device),
                     slots=torch.tensor(np.repeat(slots, new), device=device))
        args = lambda s=state: step_of(cache, s["layout"], s["lengths"], s["positions"], s["slots"], s["rows"], heads, kv_heads, rope)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            args()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = args()
        steps.append((state, args, graph, out))
    for turn in range(4):
        for state, args, graph, out in steps:
            lengths = np.array([rng.integers(n, most) for n, most in zip(new, (900, 700, 400))])
            state["lengths"].copy_(torch.from_numpy(lengths))
            state["positions"].copy_(torch.from_numpy(np.concatenate([np.arange(n) + t - n for n, t in zip(new, lengths)])))
            state["rows"].copy_(randn(rng, rows, heads + 2 * kv_heads, dim))
            cache.page_table.copy_(torch.from_numpy(table[rng.permutation(len(table))].astype(np.int32)))
            saved = cache.keys.clone(), cache.values.clone()
            graph.replay()
            first = out.clone()
            torch.cuda.synchronize()
            after = cache.keys.clone(), cache.values.clone()
            cache.keys.copy_(saved[0]), cache.values.copy_(saved[1])
            assert torch.equal(args(), first), turn
            assert torch.equal(cache.keys, after[0]) and torch.equal(cache.values, after[1])


def test_calls_on_two_streams(device):
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(19)
    lengths = [3000, 2000]
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, _, _ = cache_of(rng, device, pages, 16, 2, 128, table)
    q = [randn(rng, 2, 16, 128).to(device) for _ in range(2)]
    layout, told = layout_of(device, [0, 1, 2], slots, 1), torch.tensor(lengths, device=device)
    want = [paged_attention(x, cache, layout, told) for x in q]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for x, s, g in zip(q, streams, got):
            with torch.cuda.stream(s):
                g.append(paged_attention(x, cache, layout, told))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_cache_refusals(device):
    from drama3_amd.attention import PagedCache

    keys = torch.zeros(4, 2, 16, 64, dtype=BF16, device=device)
    values, table = torch.zeros_like(keys), torch.zeros(3, 5, dtype=torch.int32, device=device)
    one = torch.ones(2, device=device)

    def refused(error, match, *args, **kwargs):
        with pytest.raises(error, match=match):
            PagedCache(*args, **kwargs)

    PagedCache(keys, values, table)
    refused(ValueError, "device tensors", keys.cpu(), values, table)
    refused(TypeError, "bfloat16 or float8", keys.float(), values.float(), table)
    refused(TypeError, "bfloat16 or float8", keys, values.to(E4M3), table)
    refused(ValueError, "one shape", keys, values[:3], table)
    refused(ValueError, "one shape", keys[0], values[0], table)
    refused(ValueError, "power of two", keys[:, :, :12], values[:, :, :12], table)
    refused(TypeError, "int32", keys, values, table.long())
    refused(ValueError, "page_table", keys, values, table[0])
    refused(ValueError, "page_table", keys, values, table.t())
    refused(ValueError, "16 bytes", keys[..., 1:], values[..., 1:], table)
    refused(ValueError, "16 bytes", keys[..., 4:60], values[..., 4:60], table)
    refused(ValueError, "16 bytes", keys.transpose(2, 3)[..., :16], values.transpose(2, 3)[..., :16], table)
    refused(ValueError, "behind the other|overlap", keys[:1].expand(4, 2, 16, 64), values, table)
    refused(ValueError, "same memory", keys, keys, table)
    refused(ValueError, "e4m3fn caches", keys, values, table, k_scale=one)
    e_keys, e_values = keys.to(E4M3), values.to(E4M3)
    refused(TypeError, "float32", e_keys, e_values, table, k_scale=one.double())
    refused(ValueError, "contiguous", e_keys, e_values, table, v_scale=one[:1])
    refused(ValueError, "2\\^30", keys, values, torch.empty(1, (1 << 26) + 1, dtype=torch.int32, device=device))


def test_call_refusals(device):
    from drama3_amd.attention import PagedCache, Rope, append_paged, apply_rope, paged_attention, prepare_rope

    rope = prepare_rope(64, device=device)
    x = torch.zeros(5, 4, 64, dtype=BF16, device=device)
    positions = torch.arange(5, device=device)

    def refused(error, match, call, *args, **kwargs):
        with pytest.raises(error, match=match):
            call(*args, **kwargs)

    refused(ValueError, "device tensors", apply_rope, x.cpu(), positions, rope)
    refused(TypeError, "bfloat16 or float32", apply_rope, x.half(), positions, rope)
    refused(ValueError, "unit column stride", apply_rope, x.transpose(1, 2), positions, rope)
    refused(ValueError, "unit column stride", apply_rope, x[0], positions, rope)
    refused(TypeError, "int32 or int64", apply_rope, x, positions.float(), rope)
    refused(ValueError, "contiguous", apply_rope, x, positions[:4], rope)
    refused(ValueError, "rotary width", apply_rope, x[..., :32], positions, rope)
    refused(ValueError, "columns a row", apply_rope, torch.zeros(1, 2000, 64, dtype=BF16, device=device), positions[:1], rope)
    refused(TypeError, "out must be", apply_rope, x, positions, rope, out=x.float())
    refused(ValueError, "out must be", apply_rope, x, positions, rope, out=x[:4])
    refused(ValueError, "overlap", apply_rope, x[:, :2], positions, rope, out=x[:, 1:3])
    refused(ValueError, "one behind the other", apply_rope, x, positions, rope, out=x[:1].expand(5, 4, 64))
    refused(TypeError, "float64", Rope, torch.zeros(8, device=device))
    refused(ValueError, "contiguous", Rope, torch.zeros(0, dtype=torch.float64, device=device))

    cache = PagedCache.empty(4, 16, 2, 64, 3, 5, device=device)
    k = torch.zeros(5, 2, 64, dtype=BF16, device=device)
    refused(ValueError, "cache's heads", append_paged, cache, x, x, positions, positions)
    refused(ValueError, "cache's heads", append_paged, cache, k, k[:4], positions, positions)
    refused(TypeError, "bfloat16", append_paged, cache, k.float(), k.float(), positions, positions)
    refused(TypeError, "row_slots must be", append_paged, cache, k, k, positions, positions.float())
    refused(ValueError, "q must be", append_paged, cache, k, k, positions, positions, q=x[:3])
    refused(ValueError, "out goes with q", append_paged, cache, k, k, positions, positions, out=x)
    refused(ValueError, "rotary width", append_paged, cache, k, k, positions, positions, rope=prepare_rope(128, device=device))
    qkv = torch.zeros(5, 8, 64, dtype=BF16, device=device)
    refused(ValueError, "overlap", append_paged, cache, qkv[:, 4:6], qkv[:, 6:], positions, positions, q=x, out=qkv[:, 2:6])

    layout, lengths = layout_of(device, [0, 5], [0], 5), torch.tensor([5], device=device)
    refused(ValueError, "multiple of 2", paged_attention, x[:, :3], cache, layout, lengths)
    refused(ValueError, "64", paged_attention, x[..., :32], cache, layout, lengths)
    refused(TypeError, "boundaries must be int32", paged_attention, x, cache,
            type(layout)(layout.boundaries.long(), layout.sequence_slots, 5), lengths)
    refused(ValueError, "sequence_slots must be", paged_attention, x, cache, layout_of(device, [0, 2, 5], [0], 3), lengths)
    refused(TypeError, "lengths must be", paged_attention, x, cache, layout, lengths.float())
    refused(ValueError, "finite", paged_attention, x, cache, layout, lengths, scale=float("nan"))
    refused(ValueError, "window", paged_attention, x, cache, layout, lengths, window=0)
    refused(ValueError, "overlap", paged_attention, x, cache, layout, lengths, out=x)
    narrow = PagedCache.empty(4, 16, 2, 32, 3, 5, device=device)
    refused(ValueError, "head dim 32", paged_attention, x[..., :32], narrow, layout, lengths)
