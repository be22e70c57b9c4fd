"""Attention at the ends of fp32's range: scores whose spacing there is many powers
of two."""

import numpy as np
import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import BF16, E4M3, cache_of, f64, layout_of, randn, tables_for, within

pytestmark = pytest.mark.gpu


def of_equal_weights(want, sizes, most, score):
    """What a mean of `most` values of that mean size may be off by: sums in fp32 (their parts added
    up to 64 times more), a quotient, the result's half step.  Where the score is 2^23 and more (in powers
    of two) the weights are 1.  Below they are 2^e alike, e what the score's product was rounded by, and
    their rounding to bf16 multiplies the whole by at most 1 + 2^-8."""
    err = ((most + 64) * 2 * oa.F32_HALF_STEP) * sizes + 4 * oa.F32_HALF_STEP * np.abs(want)
    if score < 2.0 ** 23:
        err = err + oa.BF16_HALF_STEP * (1 + oa.BF16_HALF_STEP) * np.abs(want)
    return err + oa.BF16_HALF_STEP * (np.abs(want) + err)


# (The scores are products of two powers of two and 9, summed over a power of two of columns: exact in
# fp32 and in 64 bits, so that keys are level or far apart, whatever the scale's product is rounded to.)
@pytest.mark.parametrize("size", [96.0, 1536.0, 24576.0, 3.0 * 2 ** 29, 3.0 * 2 ** 48])
@pytest.mark.parametrize("new, lengths", [([1, 1, 1], [1, 60, 5000]), ([1, 5, 40], [1, 5, 300]), ([200, 130], [3100, 130])])
@pytest.mark.parametrize("dim, dtype", [(64, BF16), (128, BF16), (256, BF16), (128, E4M3)])
def test_scores_far_past_the_steps_of_one(device, dim, dtype, new, lengths, size):
    """Every third key's scores 1/64 below the others' (e4m3: 1/6): the softmax is the mean
    of those that share the highest, a row's only key gives its value."""
    from drama3_amd.attention import PagedCache, paged_attention

    rng = np.random.default_rng(dim + sum(lengths))
    table, slots, pages = tables_for(rng, lengths, 16)
    cache, keys, values = cache_of(rng, device, pages, 16, 2, dim, table, dtype, scales=False)
    level = torch.full((pages, 2, 16, 1), 384.0 if dtype == E4M3 else size)
    level[:, :, 1::3] = 320.0 if dtype == E4M3 else size * (1 - 1 / 64)
    cache.keys.copy_(level.expand(-1, -1, -1, dim).to(device))
    keys[...] = level.double().numpy()
    if dtype == E4M3:
        scale = torch.tensor([1.0, 3.0]) * size / 384
        cache = PagedCache(cache.keys, cache.values, cache.page_table, scale.to(device))
        keys *= f64(scale)[:, None, None]
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = torch.full((boundaries[-1], 4, dim), size, dtype=BF16)
    q[:, 1::2] *= -1  # the lower keys are theirs
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)), torch.tensor(lengths, device=device))
    with np.errstate(invalid="ignore"):
        want, _, owned = oa.attention(f64(q), keys, values, table, boundaries, slots, lengths, dim ** -0.5)
        sizes, _, _ = oa.attention(f64(q), keys, np.abs(values), table, boundaries, slots, lengths, dim ** -0.5)
    assert owned.all() and np.isfinite(want).all()
    within(out, want, of_equal_weights(want, sizes, max(lengths), size * size * dim ** 0.5 * 63 / 64))


def test_high_level_scores_of_many_rows(device):
    """Tiles of two groups of waves: all keys level, so that a row has the mean of the values up to its own."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(40)
    rows, heads, kv_heads, dim = 2100, 32, 2, 128
    table, slots, pages = tables_for(rng, [rows], 16)
    cache, _, values = cache_of(rng, device, pages, 16, kv_heads, dim, table)
    cache.keys.fill_(24576.0)
    q = torch.full((rows, heads, dim), 24576.0, dtype=BF16, device=device)
    out = paged_attention(q, cache, layout_of(device, [0, rows], slots, rows), torch.tensor([rows], device=device))
    at = np.arange(rows)
    mine = np.repeat(values[table[slots[0], at // 16], :, at % 16], heads // kv_heads, axis=1)
    count = np.arange(1, rows + 1)[:, None, None]
    want, sizes = np.cumsum(mine, 0) / count, np.cumsum(np.abs(mine), 0) / count
    within(out, want, of_equal_weights(want, sizes, rows, 24576.0 ** 2))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [None, 30])
@pytest.mark.parametrize("new, lengths", [([1, 1, 1, 1], [40, 700, 2100, 33]), ([1, 5, 140], [40, 300, 600])])
def test_scores_of_minus_infinity(device, dim, window, new, lengths):
    """Keys whose score is minus infinity weigh nothing; a row that attends only such has no softmax: NaN,
    and not the zeros of a row that attends nothing."""
    from drama3_amd.attention import paged_attention

    rng = np.random.default_rng(dim + sum(lengths))
    table, slots, pages = tables_for(rng, lengths, 1)  # (a token a page)
    cache, keys, values = cache_of(rng, device, pages, 1, 2, dim, table)
    spoiled = np.zeros(table.shape, dtype=bool)
    spoiled[slots[0], :40] = True                # the first sequence has nothing else
    spoiled[slots[1], 10:290] = True
    spoiled[slots[2], :500] = True
    table[slots[-1], lengths[-1] - 33:] = -1     # the last one's newest rows: under a window, nothing at all
    spoiled &= table >= 0
    for page in table[spoiled]:
        keys[page, :, :, 7] = -np.inf
    cache.keys.copy_(torch.from_numpy(keys).to(BF16).to(device))
    cache.page_table.copy_(torch.from_numpy(table.astype(np.int32)).to(device))
    boundaries = np.concatenate([[0], np.cumsum(new)])
    q = randn(rng, boundaries[-1], 4, dim)
    q[..., 7] = q[..., 7].abs() + 0.5
    out = paged_attention(q.to(device), cache, layout_of(device, boundaries, slots, max(new)), torch.tensor(lengths, device=device),
                          window=window)
    call = lambda t: oa.attention(f64(q), keys, values, t, boundaries, slots, lengths, dim ** -0.5, window)  # noqa: E731
    with np.errstate(all="ignore"):
        nothing = np.isnan(call(table)[0])
    want, bound, _ = call(np.where(spoiled, -1, table))
    assert nothing[0].all() and not nothing[-1].any()
    assert window is None or not want[-1].any()
    within(out, np.where(nothing, np.nan, want), bound + oa.BF16_HALF_STEP * (np.abs(want) + bound))
