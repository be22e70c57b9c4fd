"""What of two tensors' memory is shared: views of one buffer told apart element by
element, and calls whose results would lie in what they read refused (CPU only:
nothing is launched)."""

import itertools

import pytest
import torch


def elements(t):
    """Byte addresses of a tensor's elements."""
    at = {t.data_ptr()}
    for n, s in zip(t.shape, t.stride()):
        at = {a + i * s * t.element_size() for a in at for i in range(n)}
    return at


def test_views_of_a_fused_buffer_are_apart():
    from drama3_amd.attention import _meet

    buffer = torch.zeros(3, 2, 5, 4, 16, dtype=torch.bfloat16)
    keys, values = buffer[:, 0], buffer[:, 1]
    assert not _meet(keys, values) and not _meet(values, keys) and _meet(keys, keys)
    halves = torch.zeros(3, 5, 4, 32, dtype=torch.bfloat16)
    assert not _meet(halves[..., :16], halves[..., 16:]) and _meet(halves[..., :16], halves[..., 8:24])
    layers = torch.zeros(6, 3, 2, 4, 16, dtype=torch.bfloat16)
    assert not any(_meet(layers[i], layers[j]) for i, j in itertools.permutations(range(6), 2))
    by_layer = torch.zeros(3, 6, 2, 4, 16, dtype=torch.bfloat16)
    assert not any(_meet(by_layer[:, i], by_layer[:, j]) for i, j in itertools.permutations(range(6), 2))
    # (a page, a head, a token further: all but the last are shared)
    flat = torch.zeros(4 * 5 * 4 * 16, dtype=torch.bfloat16)
    for step in (16, 4 * 16, 5 * 4 * 16, 8):
        assert _meet(flat[:3 * 320].view(3, 5, 4, 16), flat[step:step + 3 * 320].view(3, 5, 4, 16))


def test_queries_and_keys_of_one_projection_are_apart():
    from drama3_amd.attention import _meet

    qkv = torch.zeros(7, 8, 16, dtype=torch.bfloat16)
    q, k, v = qkv.split((4, 2, 2), 1)
    assert not any(_meet(x, y) for x, y in itertools.permutations((q, k, v), 2))
    assert _meet(q, qkv[:, 3:5]) and _meet(qkv[:, 3:5], q)
    assert not _meet(q[2:3], k[2:3]) and not _meet(q[2:3], k) and _meet(q[2:3], qkv[:, 3:5])


@pytest.mark.parametrize("seed", range(40))
def test_sharing_is_what_the_elements_say(seed):
    """Nested strides: exactly; any others: never apart where an element is shared."""
    from drama3_amd.attention import _meet

    rng = torch.Generator().manual_seed(seed)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=rng))  # noqa: E731
    store = torch.zeros(4000, dtype=torch.uint8)
    for _ in range(50):
        columns = 1 + pick(4)
        strides, reach = [1], 4
        for _ in range(3):
            strides.insert(0, reach + pick(4))
            reach = strides[0] * (1 + pick(3))
        order = torch.randperm(3, generator=rng).tolist() + [3]
        strides = [strides[i] for i in order]
        views = []
        for _ in range(2):
            shape = [1 + pick(2), 1 + pick(2), 1 + pick(2), columns]
            mine = [s + (pick(2) if seed % 4 == 0 and n > 1 else 0) for s, n in zip(strides, shape)]
            mine[3] = 1
            views.append(store.as_strided(shape, mine, pick(60)))
        a, b = views
        shared = bool(elements(a) & elements(b))
        assert _meet(a, b) >= shared and _meet(b, a) >= shared
        def reach_of(t):  # whether each stride steps over the smaller ones
            far = 1
            for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
                if s < far:
                    return False
                far += (n - 1) * s
            return True
        alike = all(s == t or n == 1 or m == 1 for s, t, n, m in zip(a.stride(), b.stride(), a.shape, b.shape))
        if alike and seed % 4 and reach_of(a) and reach_of(b) and a.shape == b.shape:
            assert _meet(a, b) == shared == _meet(b, a)


@pytest.fixture
def launched(monkeypatch):
    """The calls' checks on tensors of the host, and what they would have launched."""
    from drama3_amd import attention

    calls = []
    monkeypatch.setattr(attention, "require_cuda", lambda *t: None)
    monkeypatch.setattr(attention, "_launch", lambda index, name, *args: calls.append(name))
    return calls


def zeros(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_keys_and_values_that_share_memory_are_refused(launched):
    from drama3_amd.attention import PagedCache

    table = torch.zeros(2, 3, dtype=torch.int32)
    page = 2 * 16 * 64
    flat = zeros(6 * page)
    view = lambda at: flat[at:at + 4 * page].view(4, 2, 16, 64)  # noqa: E731
    for step in (64, 16 * 64, page, 2 * page):  # (a token, a head, a page further)
        for pair in ((view(0), view(step)), (view(step), view(0))):
            with pytest.raises(ValueError, match="same memory"):
                PagedCache(*pair, table)
    # Of different strides within the same bytes: not told apart.
    with pytest.raises(ValueError, match="same memory"):
        PagedCache(view(0), flat[:4 * page].view(4, 16, 2, 64).transpose(1, 2), table)
    both = zeros(4, 2, 2, 16, 64)
    PagedCache(both[:, 0], both[:, 1], table)
    PagedCache(both[:, :, 0], both[:, :, 1], table)
    side = zeros(4, 2, 16, 128)
    PagedCache(side[..., :64], side[..., 64:], table)
    with pytest.raises(ValueError, match="same memory"):
        PagedCache(side[..., :64], side[..., 56:120], table)


def test_rows_within_the_cache_are_refused(launched):
    from drama3_amd.attention import PagedCache, append_paged, paged_attention
    from drama3_amd.packed_prefill import PackedLayout

    keys, values = zeros(4, 2, 16, 64), zeros(4, 2, 16, 64)
    cache = PagedCache(keys, values, torch.zeros(2, 3, dtype=torch.int32))
    at = torch.arange(5)
    k, v, q = zeros(5, 2, 64), zeros(5, 2, 64), zeros(5, 4, 64)
    inside = [t[0, :, :5].transpose(0, 1) for t in (keys, values)]
    of_queries = [t.view(-1)[-1280:].view(5, 4, 64) for t in (keys, values)]
    for bad in inside:
        with pytest.raises(ValueError, match="k must not overlap the cache"):
            append_paged(cache, bad, v, at, at)
        with pytest.raises(ValueError, match="v must not overlap the cache"):
            append_paged(cache, k, bad, at, at)
    layout = PackedLayout(torch.tensor([0, 5], dtype=torch.int32), torch.zeros(1, dtype=torch.int64), 5)
    for bad in of_queries:
        with pytest.raises(ValueError, match="q must not overlap the cache"):
            append_paged(cache, k, v, at, at, q=bad)
        with pytest.raises(ValueError, match="out must not overlap the cache"):
            append_paged(cache, k, v, at, at, q=q, out=bad)
        with pytest.raises(ValueError, match="out must not overlap the cache"):
            paged_attention(q, cache, layout, torch.tensor([5]), out=bad)
    assert not launched
    append_paged(cache, k, v, at, at, q=q)
    assert launched == ["d3_paged_append"]


def test_queries_turned_in_place_share_nothing_with_keys_and_values(launched):
    from drama3_amd.attention import PagedCache, append_paged

    cache = PagedCache(zeros(4, 2, 16, 64), zeros(4, 2, 16, 64), torch.zeros(2, 3, dtype=torch.int32))
    at = torch.arange(5)
    qkv = zeros(5, 8, 64)
    q, k, v = qkv.split((4, 2, 2), 1)
    append_paged(cache, k, v, at, at, q=q, out=q)
    append_paged(cache, k[:1], v[:1], at[:1], at[:1], q=q[:1], out=q[:1])
    assert len(launched) == 2
    for bad_k, bad_v in ((qkv[:, 3:5], v), (k, qkv[:, 2:4])):
        with pytest.raises(ValueError, match="overlap k or v"):
            append_paged(cache, bad_k, bad_v, at, at, q=q, out=q)
        append_paged(cache, bad_k, bad_v, at, at, q=q)  # (only read)
    assert len(launched) == 4
    one = zeros(1, 4, 64).as_strided((1, 4, 64), (0, 64, 1))  # (a stride that no step takes)
    append_paged(cache, one[:, :2], one[:, :2], at[:1], at[:1], q=one + 0, out=None)
    with pytest.raises(ValueError, match="overlap k or v"):
        append_paged(cache, one[:, :2], one[:, :2], at[:1], at[:1], q=one, out=one)
