"""The entry points of rotary positions, the paged cache and its attention refuse
what they cannot compute before launching anything (CPU only: no kernel is run)."""

import ctypes

import pytest

P = 1 << 20  # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    from drama3_amd import _lib

    if not _lib.LIBRARY.exists():
        pytest.skip("library not built")
    return _lib.load()


def cache(**changes):
    from drama3_amd import _lib

    fields = dict(keys=P, values=P, dtype=_lib.DTYPE_BF16, kv_heads=2, head_dim=64, page_size=16, pages=8,
                  key_page_stride=2048, key_head_stride=1024, key_token_stride=64, value_page_stride=2048,
                  value_head_stride=1024, value_token_stride=64, page_table=P, table_stride=4, slots=3, max_pages=4)
    return _lib.PagedCacheStruct(**{**fields, **changes})


def rope(**changes):
    from drama3_amd import _lib

    return _lib.RopeStruct(**{**dict(turns=P, rotary_dim=32, interleaved=0, magnitude=1.0), **changes})


def at(struct):
    return ctypes.addressof(struct) if struct is not None else None


def rope_rows(turning, **changes):
    from drama3_amd import _lib

    a = dict(x=P, dtype=0, row=256, head=64, rows=3, heads=4, dim=64, positions=P, positions_dtype=3, rope=at(turning),
             out=P, out_row=256, out_head=64)
    return _lib.call("d3_rope_rows", *{**a, **changes}.values(), None)


def append(kept, turning=None, **changes):
    from drama3_amd import _lib

    a = dict(cache=at(kept), k=P, k_row=128, k_head=64, v=P, v_row=128, v_head=64, rows=3, positions=P, positions_dtype=3,
             row_slots=P, row_slots_dtype=3, rope=at(turning), q=P, q_row=256, q_head=64, q_heads=4, q_out=P,
             q_out_row=256, q_out_head=64)
    return _lib.call("d3_paged_append", *{**a, **changes}.values(), None)


def attend(kept, **changes):
    from drama3_amd import _lib

    a = dict(cache=at(kept), q=P, q_row=256, q_head=64, rows=3, q_heads=4, boundaries=P, slots=P, slots_dtype=3, lengths=P,
             lengths_dtype=2, sequences=2, max_length=2, scale=0.125, window=0, out=2 * P, out_row=256, out_head=64,
             zero_rest=1, workspace=P, workspace_bytes=1 << 30)
    return _lib.call("d3_paged_attention", *{**a, **changes}.values(), None)


def test_rope_refusals(lib):
    turning = rope()
    with pytest.raises(ValueError, match="null rope"):
        rope_rows(None)
    with pytest.raises(ValueError, match="shape"):
        rope_rows(turning, heads=0)
    with pytest.raises(ValueError, match="shape"):
        rope_rows(turning, rows=-1)
    with pytest.raises(ValueError, match="bf16 or f32"):
        rope_rows(turning, dtype=4)
    with pytest.raises(ValueError, match="int32 or int64"):
        rope_rows(turning, positions_dtype=1)
    with pytest.raises(ValueError, match="null pointer"):
        rope_rows(turning, positions=None)
    with pytest.raises(ValueError, match="alignment"):
        rope_rows(turning, dtype=1, x=P + 2)
    with pytest.raises(ValueError, match="columns a row"):
        rope_rows(turning, heads=1025)
    with pytest.raises(ValueError, match="2\\^22 rows"):
        rope_rows(turning, rows=1 << 22)
    for changes in (dict(turns=None), dict(rotary_dim=0), dict(rotary_dim=31), dict(rotary_dim=66)):
        with pytest.raises(ValueError, match="turns|rotary width"):
            rope_rows(rope(**changes))


CACHE_FAULTS = [
    (dict(dtype=1), "bf16 or e4m3"), (dict(kv_heads=0), "shape"), (dict(pages=0), "shape"), (dict(slots=0), "shape"),
    (dict(max_pages=0), "shape"), (dict(page_size=24), "power of two"), (dict(pages=1 << 31), "2\\^31 pages"),
    (dict(max_pages=(1 << 26) + 1), "2\\^30 tokens"), (dict(key_page_stride=1 << 31), "2\\^31 elements"),
    (dict(value_head_stride=-64), "2\\^31 elements"), (dict(keys=None), "null cache pointer"),
    (dict(page_table=None), "null cache pointer"), (dict(values=P + 8), "alignment"), (dict(key_token_stride=68), "multiples"),
    (dict(dtype=4, head_dim=72), "multiples")]


@pytest.mark.parametrize("changes, match", CACHE_FAULTS)
def test_cache_refusals(lib, changes, match):
    kept = cache(**changes)
    for call in (append, attend):
        with pytest.raises(ValueError, match=match):
            call(kept)
    assert lib.d3_paged_attention_workspace(at(kept), 3, 4, 2, 2) == -1


def test_append_refusals(lib):
    kept = cache()
    with pytest.raises(ValueError, match="null cache"):
        append(None)
    with pytest.raises(ValueError, match="int32 or int64"):
        append(kept, row_slots_dtype=0)
    with pytest.raises(ValueError, match="go together"):
        append(kept, q=None)
    with pytest.raises(ValueError, match="go together"):
        append(kept, q_heads=0)
    with pytest.raises(ValueError, match="null pointer"):
        append(kept, v=None)
    with pytest.raises(ValueError, match="columns a row"):
        append(kept, q_heads=1021)
    with pytest.raises(ValueError, match="rotary width"):
        append(kept, rope(rotary_dim=128))
    with pytest.raises(ValueError, match="2\\^22 rows"):
        append(kept, rows=1 << 22)


def test_attention_refusals(lib):
    kept = cache()
    with pytest.raises(ValueError, match="null cache"):
        attend(None)
    with pytest.raises(ValueError, match="kv heads"):
        attend(kept, q_heads=3)
    with pytest.raises(ValueError, match="finite"):
        attend(kept, scale=float("inf"))
    with pytest.raises(ValueError, match="int32 or int64"):
        attend(kept, lengths_dtype=1)
    with pytest.raises(ValueError, match="head dim 32"):
        attend(cache(head_dim=32))
    with pytest.raises(ValueError, match="sequences"):
        attend(kept, sequences=65537)
    with pytest.raises(ValueError, match="rows of"):
        attend(kept, rows=(1 << 21) + 1)
    with pytest.raises(ValueError, match="null pointer"):
        attend(kept, out=None)
    with pytest.raises(ValueError, match="null pointer"):
        attend(kept, boundaries=None)
    with pytest.raises(ValueError, match="shape"):
        attend(kept, rows=-1)


@pytest.mark.parametrize("max_length", [1, 2, 64])
def test_attention_wants_its_workspace(lib, max_length):
    kept = cache(max_pages=4096)
    need = lib.d3_paged_attention_workspace(at(kept), 64, 4, 64, max_length)
    assert need > 0
    for changes in (dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=need - 1)):
        with pytest.raises(ValueError, match="workspace"):
            attend(kept, rows=64, sequences=64, max_length=max_length, **changes)


def test_calls_without_rows_touch_nothing(lib):
    kept, turning = cache(), rope()
    rope_rows(turning, rows=0, x=None, positions=None, out=None)
    append(kept, rows=0, k=None, v=None, positions=None, row_slots=None)
    attend(kept, rows=0, q=None, out=None, workspace=None, workspace_bytes=0)
    attend(kept, sequences=0, zero_rest=0, boundaries=None, slots=None, lengths=None, workspace=None, workspace_bytes=0)
    assert lib.d3_paged_attention_workspace(at(kept), 0, 4, 2, 2) == 0


@pytest.mark.parametrize("head_dim, kv_heads, q_heads", [(64, 1, 1), (128, 2, 40), (256, 4, 4)])
@pytest.mark.parametrize("max_pages", [1, 100, 1 << 26])
@pytest.mark.parametrize("rows, sequences", [(1, 1), (5, 65536), (65536, 1), (209715, 3)])
def test_workspace_stays_bounded(lib, head_dim, kv_heads, q_heads, max_pages, rows, sequences):
    """Parts are kept for what fills the card, not for the length of the sequences."""
    kept = cache(head_dim=head_dim, kv_heads=kv_heads, max_pages=max_pages)
    for max_length in (0, 1, 7, rows, 1 << 30):
        need = lib.d3_paged_attention_workspace(at(kept), rows, q_heads, sequences, max_length)
        assert 0 <= need <= 160 << 20


def test_attention_refuses_more_kv_heads_than_a_launch_holds(lib):
    """(a join takes 8,192 threads of each kv head at most: 2^29 of 65,536)"""
    wide = cache(kv_heads=65537, page_size=1, key_page_stride=65537 * 64, key_head_stride=64, value_page_stride=65537 * 64,
                 value_head_stride=64)
    with pytest.raises(ValueError, match="65537 kv heads"):
        attend(wide, rows=1, q_heads=65537, sequences=1)
    assert lib.d3_paged_attention_workspace(at(wide), 1, 65537, 1, 2) == -1


@pytest.mark.parametrize("seed", range(200))
def test_the_restated_plan_has_the_librarys_parts(lib, seed):
    """``oracle.attention.cut`` says how many partial rows a call keeps: the workspace that the library asks for."""
    import random

    from oracle import attention as oa

    rng = random.Random(seed)
    spread = lambda low, high: round(low * (high / low) ** rng.random())  # noqa: E731
    head_dim, kv_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 8, 16, 96, 700])
    q_heads = kv_heads * rng.choice([1, 2, 5, 8, 17, 40])
    rows = min(spread(1, 40000), (1 << 23) // q_heads)
    sequences = rng.choice([0, 1, spread(1, 200), spread(1, 65536)])
    max_length = rng.choice([0, 1, 2, rows, spread(1, 100000)])
    page_size = 1 << rng.randrange(9)
    max_pages = spread(1, (1 << 30) // page_size)
    kept = cache(head_dim=head_dim, kv_heads=kv_heads, page_size=page_size, max_pages=max_pages)
    # (bounds hang on the sizes alone: no sequence has a row here)
    _, most = oa.cut(rows, q_heads, kv_heads, [0] * (sequences + 1), [0] * sequences, page_size * max_pages, max_length, head_dim)
    rows_kept = (most["single_parts"] * 16 + most["tile_parts"] * most["tile_rows"]) * kv_heads
    assert lib.d3_paged_attention_workspace(at(kept), rows, q_heads, sequences, max_length) == rows_kept * (head_dim + 2) * 4


def test_attention_refuses_a_scale_that_powers_of_two_do_not_hold(lib):
    """(scores are taken times log2 e: 3e38 of it is infinite)"""
    for scale in (3e38, -3e38):
        with pytest.raises(ValueError, match="finite"):
            attend(cache(), scale=scale)
