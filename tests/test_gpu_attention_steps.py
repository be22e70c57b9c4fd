"""Steps of mixed batches by row metadata: what is added to its positions for slots
that hold tokens already."""

import numpy as np
import pytest
import torch

from test_gpu_attention import BF16, layout_of, randn

pytestmark = pytest.mark.gpu


def test_chunks_on_cached_tokens_go_behind_them(device):
    """A second chunk, a single token, a slot with no new token and a whole prompt, with rows of no
    sequence behind: each token at its own place, the others as they were."""
    from drama3_amd.attention import PagedCache, append_paged, apply_rope, paged_attention, prepare_rope
    from drama3_amd.packed_prefill import packed_row_metadata

    rng = np.random.default_rng(50)
    new, lengths, slots = [20, 1, 0, 33], [57, 40, 9, 33], [2, 0, 4, 3]
    rows, capacity, heads, kv_heads, dim = sum(new), 60, 4, 2, 64
    cache = PagedCache.empty(30, 16, kv_heads, dim, 5, 5, device=device)
    cache.page_table.copy_(torch.from_numpy(rng.permutation(30)[:25].reshape(5, 5).astype(np.int32)))
    cache.keys.normal_()
    cache.values.normal_()
    before = cache.keys.clone(), cache.values.clone()
    rope = prepare_rope(dim, device=device)
    layout = layout_of(device, np.concatenate([[0], np.cumsum(new)]), slots, max(new))
    lengths = torch.tensor(lengths, device=device)
    q, k, v = randn(rng, capacity, heads + 2 * kv_heads, dim).to(device).split((heads, kv_heads, kv_heads), 1)

    positions = torch.empty(capacity, dtype=torch.int64, device=device)
    row_slots = torch.empty_like(positions)
    packed_row_metadata(layout.boundaries, layout.sequence_slots, capacity, positions, row_slots)
    count = layout.boundaries.diff()
    positions[:rows] += torch.repeat_interleave(lengths - count, count, output_size=rows)
    row_slots[rows:] = -1

    turned = append_paged(cache, k, v, positions, row_slots, rope=rope, q=q)
    row, told, keys = 0, lengths.tolist(), apply_rope(k, positions, rope)
    wrote = torch.zeros(30, 16, dtype=torch.bool)
    for n, length, slot in zip(new, told, slots):
        for token in range(length - n, length):
            page, place = int(cache.page_table[slot, token // 16]), token % 16
            assert torch.equal(cache.keys[page, :, place], keys[row]) and torch.equal(cache.values[page, :, place], v[row])
            assert int(positions[row]) == token
            wrote[page, place] = True
            row += 1
    kept = (~wrote).to(device)[:, None, :, None]
    for store, old in zip((cache.keys, cache.values), before):
        assert torch.equal(store * kept, old * kept)
    # Each sequence by itself has the same rows.  (Cut otherwise: either is off by half a step of its weights, of values up to
    # the largest, and of itself.)
    most = float(cache.values.abs().max()) * 2 ** -7
    out = paged_attention(turned, cache, layout, lengths)
    assert not out[rows:].any() and out.dtype == BF16
    for i, (first, n) in enumerate(zip(np.cumsum([0] + new), new)):
        one = paged_attention(turned[first:first + n], cache, layout_of(device, [0, n], [slots[i]], n), lengths[i:i + 1])
        torch.testing.assert_close(one, out[first:first + n], rtol=2 ** -7, atol=most)
