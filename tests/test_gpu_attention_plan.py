"""How a call of the attention is cut: grids, shares and splits at the sizes where
they change."""

import numpy as np
import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import BF16, E4M3, cache_of, f64, layout_of, randn, reference, tables_for, within

pytestmark = pytest.mark.gpu


def test_as_many_workgroups_as_a_grid_holds(device):
    """8,191 sequences of a token and 1,024 kv heads each, where longer ones are allowed for: tiles of two groups
    of waves would be more threads than a launch has."""
    from drama3_amd.attention import PagedCache, paged_attention

    rows, heads, dim = 8191, 1024, 128
    cache = PagedCache.empty(2, 16, heads, dim, 1, 2, device=device)
    cache.keys.zero_()
    cache.values.normal_(generator=torch.Generator(device).manual_seed(3))
    cache.page_table.copy_(torch.tensor([[1, 0]]))
    lengths = torch.arange(rows, device=device) % 20 + 1
    layout = layout_of(device, np.arange(rows + 1), np.zeros(rows), 4096)
    q = torch.ones(rows + 1, heads, dim, dtype=BF16, device=device)
    full = torch.full_like(q, float("nan"))
    del full  # (the result takes its place)
    out = paged_attention(q, cache, layout, lengths)
    assert not out[rows:].any()
    values = cache.values[[1, 0]].transpose(1, 2).reshape(32, heads, dim)[:20].double()
    count = torch.arange(1, 21, device=device)[:, None, None]
    want, sizes = values.cumsum(0) / count, values.abs().cumsum(0) / count
    err = 100 * 2 * oa.F32_HALF_STEP * sizes
    bound = err + oa.BF16_HALF_STEP * (want.abs() + err)
    for first in range(0, rows, 1000):
        at = (lengths[first:first + 1000] - 1).long()
        assert ((out[first:min(first + 1000, rows)].double() - want[at]).abs() <= bound[at]).all()


def uneven(seed, count, most, chunks=0, empty=0.1):
    """(new tokens, lengths) of `count` sequences: single tokens, `chunks` of them longer, some without a
    token, some without a key."""
    rng = np.random.default_rng(seed)
    new = np.where(rng.random(count) < empty, 0, 1)
    new[rng.permutation(count)[:chunks]] = rng.integers(2, 200, chunks)
    lengths = np.maximum(new, np.exp(rng.uniform(0, np.log(most), count)).astype(int))
    lengths[rng.permutation(count)[:count // 10]] = most - rng.integers(0, 40, count // 10)
    lengths[np.flatnonzero(new == 1)[:3]] = 0
    return new, lengths


@pytest.mark.parametrize("count, chunks, heads, kv_heads, dim, window, dtype, joins, cut", [
    (100, 0, 16, 8, 128, None, BF16, "shares", False), (100, 0, 8 * 17, 8, 128, None, BF16, "shares", False),
    (100, 0, 16, 8, 128, 300, BF16, "shares", False), (160, 0, 16, 8, 64, None, BF16, "shares", False), (90, 0, 32, 8, 256, None, E4M3, "shares", False),
    (70, 0, 40, 1, 64, None, BF16, "tiles", False), (130, 0, 4, 2, 128, 700, E4M3, "tiles", False),
    (90, 12, 16, 8, 128, None, BF16, "shares", True), (90, 12, 8 * 17, 8, 64, None, BF16, "shares", False), (90, 8, 32, 8, 256, 500, BF16, "shares", False),
    (150, 20, 4, 2, 128, None, E4M3, "shares", True), (80, 5, 6, 1, 128, 900, BF16, "tiles", True)])
def test_shares_and_splits_of_more_sequences_than_a_wave(device, count, chunks, heads, kv_heads, dim, window, dtype, joins, cut):
    """More than 64 sequences, tokens whose keys several workgroups share and tiles that are cut, joined for each tile
    or, where single tokens are more than the workgroups, for each share that ends within one."""
    from drama3_amd.attention import paged_attention

    new, lengths = uneven(count + heads, count, 1500, chunks)
    rng = np.random.default_rng(count)
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, kv_heads, dim, table, dtype)
    boundaries = np.concatenate([[0], np.cumsum(new)])
    rows, longest = int(boundaries[-1]), int(new.max())
    units, most = oa.cut(rows, heads, kv_heads, boundaries, lengths, 16 * table.shape[1], longest, dim, window or 0)
    slices, group = -(-heads // kv_heads // 16), heads // kv_heads
    single_tiles = slices * (rows if longest == 1 else min(count, rows))
    assert joins == ("shares" if single_tiles > most["shares"] else "tiles")
    assert sum(u[2] and u[3] is not None for u in units) > 20  # parts of single tokens, and of tiles
    assert sum(not u[2] and u[3] is not None for u in units) > 10 or not cut
    q = randn(rng, rows, heads, dim)
    args = (q.to(device), cache, layout_of(device, boundaries, slots, longest), torch.tensor(lengths, device=device))
    out = paged_attention(*args, window=window)
    want, bound = reference(q.double().to(device), *(torch.from_numpy(t).to(device) for t in (keys, values)), table, boundaries,
                            slots, np.maximum(lengths, 1), dim ** -0.5, window)
    want, bound = f64(want), f64(bound)
    none = np.repeat(lengths == 0, new)  # (rows without a key: zeros)
    want[none], bound[none] = 0, 0
    within(out, want, bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))
    assert all(torch.equal(paged_attention(*args, window=window), out) for _ in range(3))
