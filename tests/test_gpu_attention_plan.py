"""How a call of the attention is cut: grids, shares and splits at the sizes where
they change."""

import numpy as np
import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import BF16, layout_of

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
