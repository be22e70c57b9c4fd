"""The attention oracle against other ways to the same values, the frequencies
of the rotary positions, and the bounds that the kernels' cut of a call keeps
(CPU only)."""

import math

import numpy as np
import pytest

from oracle import attention as oa


def test_rope_is_a_rotation_that_composes():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 3, 16))
    f = 10000.0 ** (-np.arange(4) / 4)
    p, r = rng.integers(0, 1000, 5), rng.integers(0, 1000, 5)
    for interleaved in (False, True):
        once, _ = oa.rope(x, p + r, f, interleaved=interleaved)
        twice, _ = oa.rope(oa.rope(x, p, f, interleaved=interleaved)[0], r, f, interleaved=interleaved)
        assert np.allclose(once, twice, atol=1e-12)
        assert np.allclose((once ** 2).sum(-1), (x ** 2).sum(-1))
        assert np.array_equal(once[..., 8:], x[..., 8:])


def test_rope_layouts_are_a_permutation_of_each_other():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 2, 12))
    f = 100.0 ** (-np.arange(6) / 6)
    p = np.arange(4) * 7
    order = np.arange(12).reshape(2, 6).T.ravel()  # half layout's columns in pair order
    half, _ = oa.rope(x, p, f)
    assert np.allclose(oa.rope(x[..., order], p, f, interleaved=True)[0], half[..., order])


def test_rope_frequencies():
    from drama3_amd.attention import rope_frequencies

    plain = rope_frequencies(8, base=10000.0)
    assert np.allclose(plain, [1.0, 0.1, 0.01, 0.001])
    assert np.allclose(rope_frequencies(8, scaling="linear", factor=4.0), np.array(plain) / 4)
    grown = rope_frequencies(8, scaling="base", factor=4.0)
    assert grown[0] == 1.0 and math.isclose(grown[-1], plain[-1] / 4)  # the slowest as under "linear"
    bands = rope_frequencies(128, scaling="bands", factor=4.0, original_length=4096)
    every = rope_frequencies(128)
    turns = 4096 * np.array(every) / (2 * math.pi)
    assert all(b == f for b, f, t in zip(bands, every, turns) if t >= 32)
    assert all(math.isclose(b, f / 4) for b, f, t in zip(bands, every, turns) if t <= 1)
    between = [(b, f) for b, f, t in zip(bands, every, turns) if 1 < t < 32]
    assert between and all(f / 4 < b < f for b, f in between)


@pytest.mark.parametrize("kwargs, error", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(rotary_dim=8, scaling="other"), "none of"),
    (dict(rotary_dim=8, base=0.0), "positive"), (dict(rotary_dim=8, scaling="linear", factor=-1.0), "positive"),
    (dict(rotary_dim=8, scaling="bands", factor=2.0), "original length"),
    (dict(rotary_dim=8, scaling="bands", factor=2.0, original_length=64, slow=4.0, fast=2.0), "slow < fast")])
def test_rope_frequency_refusals(kwargs, error):
    from drama3_amd.attention import rope_frequencies

    with pytest.raises(ValueError, match=error):
        rope_frequencies(**kwargs)


def test_e4m3_rounding_is_the_types_own():
    import torch

    rng = np.random.default_rng(2)
    x = np.concatenate([rng.standard_normal(4000) * np.exp(3 * rng.standard_normal(4000)),
                        np.arange(-512, 513) / 64.0, np.arange(-64, 65) * 2.0 ** -10, [448.0, 460.0, -1e9]])
    # (values that fp32 holds: torch's conversion goes through it)
    x = x.astype(np.float32).astype(np.float64)
    want = torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(oa.e4m3(x), want)


def test_attention_over_pages_is_attention_over_rows():
    rng = np.random.default_rng(3)
    page_size, kv_heads, dim = 4, 2, 8
    keys, values = rng.standard_normal((2, 9, kv_heads, page_size, dim))
    table = np.array([[3, 7, -1, 1], [0, 8, 2, 99]])
    q = rng.standard_normal((6, 4, dim))
    out, bound, owned = oa.attention(q, keys, values, table, [1, 4, 4, 5], [0, 1, 1], [10, 7, 16], 0.5, window=6)
    assert owned.tolist() == [False, True, True, True, True, False]
    for row, slot, position in ((1, 0, 7), (2, 0, 8), (3, 0, 9), (4, 1, 15)):
        for head in range(4):
            k = [(table[slot, t // 4], t % 4) for t in range(max(0, position - 5), position + 1)]
            k = [(p, t) for p, t in k if 0 <= p < 9]
            s = np.array([0.5 * q[row, head] @ keys[p, head // 2, t] for p, t in k])
            w = np.exp(s) / np.exp(s).sum()
            assert np.allclose(out[row, head], w @ np.array([values[p, head // 2, t] for p, t in k]))
    assert (bound[owned] > 0).all() and not out[~owned].any()


@pytest.mark.parametrize("seed", range(60))
def test_cut_covers_every_row_and_key_within_its_bounds(seed):
    """The unit list that the kernels derive: as many as the grid holds, partials
    within the workspace, every tile's keys partitioned by its splits."""
    rng = np.random.default_rng(seed)
    kv_heads = int(rng.choice([1, 2, 4, 8, 16, 96]))
    q_heads = kv_heads * int(rng.choice([1, 2, 3, 5, 8, 16, 17, 24, 40]))
    count = int(rng.integers(1, 70))
    decode = seed % 2 == 0
    tokens = rng.integers(0, 2, count) if decode else (np.exp(rng.uniform(0, 5.5, count)) * rng.integers(0, 2, count)).astype(int)
    boundaries = np.concatenate([[0], tokens.cumsum()]) + int(rng.integers(0, 3))
    rows = int(boundaries[-1] + rng.integers(0, 4))
    if rows == 0:
        return
    capacity = 16 * int(np.exp(rng.uniform(0, 8)))
    lengths = tokens + (np.exp(rng.uniform(0, np.log(capacity + 1), count)) - 2).astype(int)
    window = int(rng.choice([0, 0, 1, 100, 1000]))
    group = q_heads // kv_heads
    dim = int(rng.choice([64, 128, 256]))
    units, most = oa.cut(rows, q_heads, kv_heads, boundaries, lengths, capacity, 1 if decode else int(tokens.max()), dim, window)
    tiles = [u for u in units if not u[2]]
    assert len(tiles) <= most["tile_units"] and -(-most["total"] // most["each"]) <= most["shares"]
    for name, mine in (("tile_parts", tiles), ("single_parts", [u for u in units if u[2]])):
        parts = [u[3] for u in mine if u[3] is not None]
        assert len(set(parts)) == len(parts) and all(0 <= p < most[name] for p in parts)
    assert len({u[:2] for u in tiles if u[3] is not None}) <= most["split_tiles"]
    for i in range(count):
        seen = []
        for tile in {u[1] for u in units if u[0] == i}:
            mine = [u for u in units if u[:2] == (i, tile)]
            start, end = mine[0][5]
            at = start
            for u in mine:  # consecutive ranges, cut at whole blocks, parts where the join looks for them
                low, high = u[4]
                if low < high:
                    assert low == at and (low == start or low % oa.BLOCK == 0)
                    at = high
                n = mine.index(u)
                assert u[3] is None or u[3] == mine[0][3] + (2 * n - (n > 0) if u[2] else n)
            assert at == end and (len(mine) == 1) == (mine[0][3] is None)
            seen += range(mine[0][6][0], mine[0][6][1] + 1)
        assert sorted(seen) == list(range(tokens[i] * group))


def test_tiles_are_split_into_as_many_units_as_are_aimed_at():
    """The blocks of a batch over the units aimed at, in integers: 8 tiles of 1,024 blocks are 512
    units of 16, not 488 of 17 by a sum that rounds."""
    units, most = oa.cut(1024, 1, 1, [0, 1024], [65536], 65536, 1024)
    assert len(units) == most["tile_units"] - 1 - 8 == 512
    assert {high - low for _, tile, _, _, (low, high), _, _ in units if tile == 7} == {1024}


@pytest.mark.parametrize("seed", range(8))
def test_cut_of_the_largest_tables_stays_within_its_bounds(seed):
    """Sums of blocks past 32 bits: tables of 2^30 tokens."""
    rng = np.random.default_rng(seed)
    count = 3000
    tokens = rng.integers(0, 4, count)
    boundaries = np.concatenate([[0], tokens.cumsum()])
    lengths = (1 << 30) - rng.integers(0, 1 << 28, count)
    group = 40
    units, most = oa.cut(int(boundaries[-1]), group, 1, boundaries, lengths, 1 << 30, 4, 128)
    tiles = [u for u in units if not u[2]]
    assert len(tiles) <= most["tile_units"]
    parts = [u[3] for u in tiles if u[3] is not None]
    assert len(set(parts)) == len(parts) and max(parts, default=-1) < most["tile_parts"]
    assert len({u[:2] for u in tiles if u[3] is not None}) <= most["split_tiles"]
