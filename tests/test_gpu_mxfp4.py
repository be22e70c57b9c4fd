"""The MXFP4 operators against the 64-bit oracle: quantised bytes exactly, the
products within the bound an fp32 evaluation has (derived in the oracle), at
the sizes, strides, boundaries and ids where they can go wrong."""

import numpy as np
import pytest
import torch

from oracle import mxfp4 as om

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def rows_of(rng, rows, width, spread=0.5):
    x = rng.standard_normal((rows, width)) * np.exp(spread * rng.standard_normal((rows, 1)))
    x *= np.exp(spread * rng.standard_normal(width))
    return torch.from_numpy(x).to(torch.bfloat16)


def weight_of(rng, *shape):
    """Random codes and scales [.., N, K] and the values they stand for."""
    w = rng.standard_normal(shape) * shape[-1] ** -0.5 * np.exp(0.5 * rng.standard_normal((*shape[:-1], 1)))
    codes, scales = om.quantize(w)
    return torch.from_numpy(codes), torch.from_numpy(scales), om.dequantize(codes, scales)


def within(got, want, bound):
    """Every element within its bound; NaN exactly where the oracle has it."""
    got = f64(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    live = ~np.isnan(want)
    excess = np.abs(got - want)[live] - bound[live]
    assert (excess <= 0).all(), f"{(excess > 0).sum()} of {excess.size} beyond, worst by {excess.max()}"


def product(x, values):
    """The oracle's product of quantised bf16 rows, and what bf16 results may be off by."""
    y, err = om.product(om.dequantize(*om.quantize(f64(x))), values)
    return y, err + om.BF16_HALF_STEP * (np.abs(y) + err)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, width", [(1, 32), (1, 2048), (3, 96), (7, 160), (257, 416), (33, 2048)])
def test_quantized_bytes(device, rows, width, dtype):
    from drama3_amd.mxfp4 import quantize_mxfp4

    rng = np.random.default_rng(rows * 10000 + width)
    x = torch.from_numpy(rng.standard_normal((rows, width)) * np.exp(6 * rng.standard_normal((rows, 1)))).to(dtype)
    x[0, :32] = 0
    codes, scales = quantize_mxfp4(x.to(device))
    want_codes, want_scales = om.quantize(f64(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantized_bytes_of_any_bit_pattern(device, dtype):
    """Subnormals, the largest magnitudes, infinities, NaN: blocks of values of
    one binade and of random patterns, whole rows of ties."""
    from drama3_amd.mxfp4 import quantize_mxfp4

    rng = np.random.default_rng(11)
    if dtype == torch.bfloat16:
        bits = rng.integers(0, 1 << 16, (4096, 64), dtype=np.uint16)
        bits[:2048] = (bits[:2048] & 0x807f) | (rng.integers(0, 256, (2048, 1), dtype=np.uint16) << 7)
        x = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16)
    else:
        bits = rng.integers(0, 1 << 32, (4096, 64), dtype=np.uint32)
        bits[:2048] = (bits[:2048] & 0x807fffff) | (rng.integers(0, 256, (2048, 1), dtype=np.uint32) << 23)
        x = torch.from_numpy(bits.view(np.int32)).view(torch.float32)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 8).to(dtype)
    x[2048:2304] = ties * torch.exp2(torch.arange(-130, 126).to(torch.float32))[:, None].to(dtype) * torch.tensor(
        [1, -1] * 32).to(dtype)
    codes, scales = quantize_mxfp4(x.to(device))
    want_codes, want_scales = om.quantize(f64(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)


def test_quantize_strided_rows_at_odd_addresses(device):
    from drama3_amd.mxfp4 import quantize_mxfp4

    rng = np.random.default_rng(12)
    wide = rows_of(rng, 40, 301)
    for first, width, step in ((0, 96, 1), (1, 128, 2), (3, 288, 1), (0, 32, 40)):
        x = wide[::step, first:first + width]
        codes, scales = quantize_mxfp4(wide.to(device)[::step, first:first + width])
        want_codes, want_scales = om.quantize(f64(x))
        assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), want_scales)
    one = wide[:1, :64].to(device).expand(5, 64)  # a row stride of zero
    codes, _ = quantize_mxfp4(one)
    assert torch.equal(codes, codes[:1].expand(5, 32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_code_at_every_scale_reads_as_its_value(device, dtype):
    from drama3_amd.mxfp4 import dequantize_mxfp4

    nibble = np.arange(16, dtype=np.uint8)
    codes = np.tile((nibble | (nibble[::-1] << 4)), (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    got = f64(dequantize_mxfp4(torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device), dtype))
    want = om.dequantize(codes, scales)
    want[np.abs(want) > float(torch.finfo(torch.float32).max)] *= np.inf  # 4 and 6 at scale 2^126 and 2^127
    assert np.array_equal(got, want, equal_nan=True)


def test_quantize_and_back_past_32_bit_offsets(device):
    """Rows beyond 2^31 elements, 2^32 bytes: the last rows are the oracle's."""
    from drama3_amd.mxfp4 import dequantize_mxfp4, quantize_mxfp4

    rows, width = 1_100_003, 4096
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device=device)
    tail = rows_of(np.random.default_rng(13), 5, width)
    x[-5:] = tail.to(device)
    codes, scales = quantize_mxfp4(x)
    want_codes, want_scales = om.quantize(f64(tail))
    assert np.array_equal(codes[-5:].cpu().numpy(), want_codes)
    assert np.array_equal(scales[-5:].cpu().numpy(), want_scales)
    assert not codes[-6].any() and not scales[-6].any()
    del x
    values = dequantize_mxfp4(codes, scales)
    assert np.array_equal(f64(values[-5:]), om.dequantize(want_codes, want_scales))
    assert not values[-6].any()


def test_quantize_more_units_than_32_bits_count(device):
    """2^32 runs of eight elements and a few more, the same row all along."""
    from drama3_amd.mxfp4 import quantize_mxfp4

    x = rows_of(np.random.default_rng(28), 1, 32)
    rows = (1 << 30) + 5
    codes, scales = quantize_mxfp4(x.to(device).expand(rows, 32))
    want_codes, want_scales = om.quantize(f64(x))
    for part in (slice(0, 3), slice((1 << 29) - 2, (1 << 29) + 2), slice(rows - 8, rows)):
        assert (codes[part].cpu().numpy() == want_codes).all() and (scales[part].cpu().numpy() == want_scales).all()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 33, 64, 65, 127, 129, 300])
@pytest.mark.parametrize("k, n", [(128, 1), (256, 64), (384, 33), (1152, 200)])
def test_linear(device, rows, k, n):
    from drama3_amd.mxfp4 import mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(rows * 7919 + k + n)
    x = rows_of(rng, rows, k)
    codes, scales, values = weight_of(rng, n, k)
    out = mxfp4_linear(x.to(device), prepare_mxfp4(codes.to(device), scales.to(device)))
    assert out.dtype == torch.bfloat16
    within(out, *product(x, values))


@pytest.mark.parametrize("rows, k, n", [(1, 2048, 1281), (52, 2048, 1281), (1030, 512, 1281), (2500, 256, 700)])
def test_linear_of_the_projection(device, rows, k, n):
    from drama3_amd.mxfp4 import mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(rows + n)
    x = rows_of(rng, rows, k)
    codes, scales, values = weight_of(rng, n, k)
    within(mxfp4_linear(x.to(device), prepare_mxfp4(codes.to(device), scales.to(device))), *product(x, values))


@pytest.mark.parametrize("rows, k, n", [
    (600, 384, 1500),                                                                # streamed, 32 rows an item
    (1000, 384, 1500), (831, 640, 1500),                                             # tiles of 32 rows
    (2100, 384, 1500), (2049, 128, 1601), (2111, 256, 1500),                         # items of 64, the last of 52, 1, 63
    (4200, 384, 1500), (4097, 128, 1537), (4136, 640, 1500), (4166, 1152, 1409)])    # of 128, the last of 104, 1, 40, 70
def test_linear_of_many_rows(device, rows, k, n):
    """Items of every size, their last ones in bodies of one to four tiles, K
    an odd and an even number of half steps; every other row of a wider buffer."""
    from drama3_amd.mxfp4 import mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(rows + k + n)
    x = rows_of(rng, rows, k)
    x[rows - 2, k - 1] = float("nan")
    codes, scales, values = weight_of(rng, n, k)
    weight = prepare_mxfp4(codes.to(device), scales.to(device))
    wide = torch.zeros((2 * rows, k + 3), dtype=torch.bfloat16, device=device)
    wide[::2, 1:k + 1] = x.to(device)
    out = mxfp4_linear(x.to(device), weight)
    within(out, *product(x, values))
    assert torch.equal(mxfp4_linear(wide[::2, 1:k + 1], weight).nan_to_num(9), out.nan_to_num(9))


def test_linear_takes_any_rows_and_keeps_nan_in_its_row(device):
    """Strided rows at odd addresses; a row with an infinity or a NaN is NaN,
    its neighbours are not (K an odd multiple of 128: the padded half step lies
    in the next row)."""
    from drama3_amd.mxfp4 import mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(14)
    for k in (128, 384, 512):
        wide = rows_of(rng, 60, k + 7)
        wide[5, 3], wide[6, k - 1], wide[40, 64] = float("inf"), float("nan"), float("-inf")
        codes, scales, values = weight_of(rng, 48, k)
        weight = prepare_mxfp4(codes.to(device), scales.to(device))
        for x in (wide[:, :k], wide[::3, 1:k + 1], wide[4:8, 3:k + 3]):
            # a view of the device copy with the same strides
            on = torch.as_strided(wide.to(device), x.shape, x.stride(), x.storage_offset())
            with np.errstate(invalid="ignore"):
                want, bound = product(x, values)
            within(mxfp4_linear(on, weight), want, bound)


def test_weights_with_nan_scales_and_extremes(device):
    from drama3_amd.mxfp4 import mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(15)
    x = rows_of(rng, 9, 256)
    codes, scales, _ = weight_of(rng, 70, 256)
    scales[3, 1], scales[69, 7], scales[10], scales[11] = 255, 255, 0, 250
    codes[11] &= 0x11  # at most 1/2: no overflow of the fp32 sums
    values = om.dequantize(codes.numpy(), scales.numpy())
    out = mxfp4_linear(x.to(device), prepare_mxfp4(codes.to(device), scales.to(device)))
    want, bound = product(x, values)
    assert np.isnan(want[:, 3]).all() and np.isfinite(want[:, 11]).all()
    within(out, want, bound + 2.0 ** -133)  # row 10's results: bf16 subnormals, a step of 2^-133


# ---------------------------------------------------------------------------
GROUPS = [
    [0, 5, 5, 5, 40, 41, 100],            # empty groups, one row, several tiles
    [0, 0, 0, 0, 0, 0, 100],              # one group holds every row
    [0, 16, 32, 48, 64, 80, 96],          # whole tiles, four rows of no group
    [7, 20, 33, 34, 50, 50, 91],          # rows of no group on both sides
    [0, 0, 0, 0, 0, 0, 0],                # no group at all
    [100, 100, 100, 100, 100, 100, 100],
    [-3, 10, 20, 30, 40, 90, 2_000_000],  # clamped to the rows there are
]


def grouped_oracle(x, bounds, values):
    want, bound = np.zeros((len(x), values.shape[1])), np.zeros((len(x), values.shape[1]))
    live = np.zeros(len(x), dtype=bool)
    ends = np.clip(bounds, 0, len(x))
    for e in range(len(values)):
        a, b = ends[e], ends[e + 1]
        if b > a:
            want[a:b], bound[a:b] = product(x[a:b], values[e])
            live[a:b] = True
    return want, bound, live


@pytest.mark.parametrize("bounds", GROUPS)
@pytest.mark.parametrize("k, n", [(256, 96), (640, 50)])
def test_grouped(device, bounds, k, n):
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    rng = np.random.default_rng(sum(bounds) + n)
    x = rows_of(rng, 100, k)
    codes, scales, values = weight_of(rng, 6, n, k)
    weight = prepare_mxfp4(codes.to(device), scales.to(device))
    boundaries = torch.tensor(bounds, dtype=torch.int32, device=device)
    want, bound, live = grouped_oracle(x, bounds, values)
    out = grouped_mxfp4(x.to(device), boundaries, weight)
    within(out, want, bound)
    assert not out[~torch.from_numpy(live).to(device)].any()
    # a given out, a column slice of a wider buffer: only the groups' rows change
    buffer = torch.full((100, n + 9), -3.0, dtype=torch.bfloat16, device=device)
    given = grouped_mxfp4(x.to(device), boundaries, weight, out=buffer[:, 5:5 + n])
    assert torch.equal(given, torch.where(torch.from_numpy(live).to(device)[:, None], out, -3.0))
    assert (buffer[:, :5] == -3).all() and (buffer[:, 5 + n:] == -3).all()


@pytest.mark.parametrize("rows, experts, k, n", [(700, 3, 128, 1000), (3000, 16, 256, 64), (900, 100, 256, 130),
                                                 (4000, 2000, 128, 40), (1, 5, 384, 65),
                                                 (48, 1, 384, 130), (49, 1, 384, 130)])
def test_grouped_at_random(device, rows, experts, k, n):
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    rng = np.random.default_rng(rows + experts)
    x = rows_of(rng, rows, k)
    codes, scales, values = weight_of(rng, experts, n, k)
    share = rng.dirichlet(np.full(experts, 0.3))
    bounds = np.concatenate([[0], np.cumsum(rng.multinomial(rows - rows // 20, share))])
    out = grouped_mxfp4(x.to(device), torch.from_numpy(bounds.astype(np.int32)).to(device),
                        prepare_mxfp4(codes.to(device), scales.to(device)))
    want, bound, _ = grouped_oracle(x, bounds, values)
    within(out, want, bound)


RAGGED = {  # groups that fill one to four tiles of an item, whole items, a row more, none
    300: [2, 2, 35, 100, 101, 165, 299],
    2100: [3, 36, 36, 133, 262, 263, 2090],
}


@pytest.mark.parametrize("rows, k, n", [(300, 384, 6500), (300, 640, 8301), (2100, 256, 8301)])
def test_grouped_over_many_columns(device, rows, k, n):
    """Items of 64 and 128 rows of ragged groups; the last case's results are
    more than the L2s hold.  Odd columns, into a column slice of a wider buffer."""
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    rng = np.random.default_rng(rows + k + n)
    bounds = RAGGED[rows]
    x = rows_of(rng, rows, k)
    codes, scales, values = weight_of(rng, 6, n, k)
    weight = prepare_mxfp4(codes.to(device), scales.to(device))
    boundaries = torch.tensor(bounds, dtype=torch.int32, device=device)
    want, bound, live = grouped_oracle(x, bounds, values)
    out = grouped_mxfp4(x.to(device), boundaries, weight)
    within(out, want, bound)
    live = torch.from_numpy(live).to(device)
    assert not out[~live].any()
    buffer = torch.full((rows, n + 10), -3.0, dtype=torch.bfloat16, device=device)
    given = grouped_mxfp4(x.to(device), boundaries, weight, out=buffer[:, 5:5 + n])
    assert torch.equal(given, torch.where(live[:, None], out, -3.0))
    assert (buffer[:, :5] == -3).all() and (buffer[:, 5 + n:] == -3).all()


@pytest.mark.parametrize("rows", [512, 513])
def test_grouped_with_one_busy_group(device, rows):
    """Most rows of many groups that one launch walks, and one row more."""
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    rng = np.random.default_rng(rows)
    x = rows_of(rng, rows, 384)
    codes, scales, values = weight_of(rng, 100, 130, 384)
    bounds = np.concatenate([np.minimum(np.arange(50), 20), np.full(51, rows - 7)])
    bounds[60:] += np.minimum(np.arange(41), 6)
    out = grouped_mxfp4(x.to(device), torch.from_numpy(bounds.astype(np.int32)).to(device),
                        prepare_mxfp4(codes.to(device), scales.to(device)))
    want, bound, _ = grouped_oracle(x, bounds, values)
    within(out, want, bound)


def test_grouped_weights_past_32_bit_offsets(device):
    """More than 4 GiB of packed codes: the last expert is found."""
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    experts, n, k = 530, 4096, 4096
    codes = torch.zeros((experts, n, k // 2), dtype=torch.uint8, device=device)
    scales = torch.full((experts, n, k // 32), 127, dtype=torch.uint8, device=device)
    rng = np.random.default_rng(16)
    last_codes, last_scales, values = weight_of(rng, n, k)
    codes[-1], scales[-1] = last_codes.to(device), last_scales.to(device)
    weight = prepare_mxfp4(codes, scales)
    del codes
    x = rows_of(rng, 20, k)
    bounds = torch.full((experts + 1,), 3, dtype=torch.int32, device=device)
    bounds[0], bounds[-1] = 0, 20
    out = grouped_mxfp4(x.to(device), bounds, weight)
    assert not out[:3].any()
    want, bound = product(x[3:], values)
    within(out[3:], want, bound)


# ---------------------------------------------------------------------------
def make_experts(rng, experts, hidden, inter, device):
    from drama3_amd.mxfp4 import prepare_mxfp4_experts

    c13, s13, v13 = weight_of(rng, experts, 2 * inter, hidden)
    c2, s2, v2 = weight_of(rng, experts, hidden, inter)
    packed = prepare_mxfp4_experts(*(t.to(device) for t in (c13, s13, c2, s2)))
    return packed, v13, v2


def make_routes(rng, rows, experts, top_k, skew=0.0):
    logits = rng.standard_normal((rows, experts)) + skew * rng.standard_normal(experts)
    ids = np.argsort(-logits, 1)[:, :top_k]
    weights = np.exp(np.take_along_axis(logits, ids, 1))
    return torch.from_numpy(ids.copy()), torch.from_numpy(weights / weights.sum(1, keepdims=True))


@pytest.mark.parametrize("rows, experts, hidden, inter, top_k, skew", [
    (1, 16, 256, 128, 8, 0), (1, 1, 128, 128, 1, 0), (5, 60, 384, 256, 8, 0), (40, 16, 256, 384, 4, 1.5),
    (130, 8, 512, 128, 2, 0), (64, 200, 256, 128, 8, 0), (300, 4, 128, 256, 1, 1.0), (17, 16, 640, 128, 16, 0),
    (600, 8, 256, 256, 8, 0.8), (3, 4, 2304, 256, 2, 0), (40, 4, 2304, 128, 8, 0), (30, 512, 128, 128, 5, 0)])
def test_moe(device, rows, experts, hidden, inter, top_k, skew):
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(rows * 31 + experts)
    packed, v13, v2 = make_experts(rng, experts, hidden, inter, device)
    x = rows_of(rng, rows, hidden)
    ids, weights = make_routes(rng, rows, experts, top_k, skew)
    weights = weights.to(torch.bfloat16)
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    within(out, *om.moe(f64(x), ids.numpy(), f64(weights), v13, v2))


@pytest.mark.parametrize("rows, experts, top_k, inter, id_type", [
    (32, 3, 4, 1152, torch.int32), (129, 3, 1, 128, torch.int32), (43, 512, 3, 128, torch.int64), (320, 5, 4, 128, torch.int32),
    (427, 5, 3, 128, torch.int64), (40, 200, 8, 640, torch.int32), (150, 200, 8, 640, torch.int64)])
def test_moe_pairs_found_by_their_experts(device, rows, experts, top_k, inter, id_type):
    """Batches without a sort (up to 1280 pairs of few workgroups) and with one:
    all pairs of one expert (the last of them), of two, every count around whole
    tiles, ids of no expert."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(rows + experts)
    packed, v13, v2 = make_experts(rng, experts, 128, inter, device)
    x = rows_of(rng, rows, 128)
    pairs = rows * top_k
    weights = torch.from_numpy(rng.random((rows, top_k))).to(torch.bfloat16)
    last = experts - 1
    patterns = [np.full(pairs, last), np.where(np.arange(pairs) < 65, last, 0), np.where(np.arange(pairs) % 17, last, 0),
                np.repeat(np.arange(-1, pairs // 16 + 1), 17)[:pairs] % (experts + 1),
                np.repeat(np.arange(pairs // 15 + 1), 16)[:pairs] % experts - 1, np.full(pairs, experts),
                rng.integers(-2, experts + 2, pairs)]
    for ids in patterns:
        ids = torch.from_numpy(rng.permutation(ids).reshape(rows, top_k)).to(id_type)
        out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
        within(out, *om.moe(f64(x), ids.numpy(), f64(weights), v13, v2))


@pytest.mark.parametrize("rows, hidden, inter, skew", [(150, 640, 1152, 0.5), (320, 384, 1024, 0.0),
                                                       (330, 256, 1152, 1.0)])
def test_moe_in_large_items(device, rows, hidden, inter, skew):
    """Items of 64 and of 128 rows in both products, their last ones of any
    size; widths of whole and half steps; rows that are NaN keep to themselves."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(rows + hidden)
    packed, v13, v2 = make_experts(rng, 8, hidden, inter, device)
    x = rows_of(rng, rows, hidden)
    ids, weights = make_routes(rng, rows, 8, 8, skew)
    ids[rng.random(ids.shape) < 0.3] = 8  # no expert: groups of different sizes
    ids, weights = ids.to(torch.int32), weights.to(torch.bfloat16)
    clean = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    within(clean, *om.moe(f64(x), ids.numpy(), f64(weights), v13, v2))
    ids[7, 0] = ids[rows - 1, 3] = 1
    x[7, 1], x[rows - 1, hidden - 1] = float("inf"), float("nan")
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    assert out[7].isnan().all() and out[-1].isnan().all()
    keep = [r for r in range(rows - 1) if r != 7]
    assert torch.equal(out[keep], clean[keep])


def test_moe_rows_past_32_bit_offsets(device):
    """Gathered rows whose offsets pass 2^31, routes' rows past 2^32 elements."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(25)
    rows, hidden = 4_500_001, 1024
    packed, v13, v2 = make_experts(rng, 2, hidden, 128, device)
    x = torch.zeros((rows, hidden), dtype=torch.bfloat16, device=device)
    tail = rows_of(rng, 40, hidden)
    x[-40:] = tail.to(device)
    ids = torch.zeros((rows, 1), dtype=torch.int32, device=device)
    ids[-25:] = 1
    weights = torch.full((rows, 1), 0.5, device=device)
    out = mxfp4_moe(x, ids, weights, packed)
    assert not out[:-40].any()
    within(out[-40:], *om.moe(f64(tail), ids[-40:].cpu().numpy(), f64(weights[-40:]), v13, v2))


@pytest.mark.parametrize("id_type, weight_type", [(torch.int32, torch.float32), (torch.int64, torch.bfloat16)])
def test_moe_ids_that_name_no_expert_add_nothing(device, id_type, weight_type):
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(17)
    packed, v13, v2 = make_experts(rng, 12, 256, 128, device)
    x = rows_of(rng, 50, 256 + 3)[:, 3:]
    ids, weights = make_routes(rng, 50, 12, 4)
    ids[0], ids[1, 2], ids[2, :] = -1, 12, torch.tensor([3, 3, 3, 99])
    ids[7, 0] = 2 ** 31 - 1
    weights[1, 2] = float("nan")  # of a rank that adds nothing
    weights[3, 1] = 0.0
    ids, weights = ids.to(id_type), weights.to(weight_type)
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    assert not out[0].any()
    within(out, *om.moe(f64(x), ids.numpy(), f64(weights), v13, v2))


def test_moe_repeated_experts_and_nan_rows(device):
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(18)
    packed, v13, v2 = make_experts(rng, 4, 384, 128, device)
    x = rows_of(rng, 33, 384)
    ids = torch.zeros((33, 3), dtype=torch.int64)
    ids[20:] = 2
    weights = torch.rand((33, 3), generator=torch.Generator().manual_seed(1))
    clean = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    within(clean, *om.moe(f64(x), ids.numpy(), f64(weights), v13, v2))
    x[4, 100], x[25, 383] = float("nan"), float("inf")
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    assert out[4].isnan().all() and out[25].isnan().all()
    keep = [r for r in range(33) if r not in (4, 25)]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("rows, id_type", [(1000, torch.int32), (1500, torch.int64), (8192, torch.int32),
                                           (9000, torch.int64)])
def test_moe_many_pairs(device, rows, id_type):
    """More pairs than one workgroup has threads, than it groups, and than
    workgroups by chunk do; now and then an id that names no expert."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(19)
    packed, v13, v2 = make_experts(rng, 24, 128, 128, device)
    x = rows_of(rng, rows, 128)
    ids, weights = make_routes(rng, rows, 24, 8, 0.7)
    ids[rng.random(ids.shape) < 0.02] = -5
    ids, weights = ids.to(id_type), weights.to(torch.bfloat16)
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    pick = rng.choice(rows, 150, replace=False)
    want, bound = om.moe(f64(x)[pick], ids.numpy()[pick], f64(weights)[pick], v13, v2)
    within(out[torch.from_numpy(pick).to(device)], want, bound)


def test_a_row_does_not_depend_on_its_batch(device):
    """The same row alone, in a handful and in a large batch: the products'
    sums may be split differently, so within two bf16 steps; the same call
    twice: the same bits."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(20)
    packed, v13, v2 = make_experts(rng, 16, 512, 256, device)
    x = rows_of(rng, 400, 512)
    ids, weights = make_routes(rng, 400, 16, 8)
    on = [t.to(device) for t in (x, ids, weights.to(torch.float32))]
    large = mxfp4_moe(*on, packed)
    assert torch.equal(large, mxfp4_moe(*on, packed))
    want, bound = om.moe(f64(x[:3]), ids.numpy()[:3], f64(on[2][:3]), v13, v2)
    within(large[:3], want, bound)
    within(mxfp4_moe(*(t[:3] for t in on), packed), want, bound)
    within(mxfp4_moe(*(t[:1] for t in on), packed), want[:1], bound[:1])


# ---------------------------------------------------------------------------
def test_operators_take_mxfp4_experts(device):
    """From FP8 experts to MXFP4 ones, and through the framework's MoE entry
    points: routing, routed experts, the reserved-padding router."""
    from drama3_amd import workloads
    from drama3_amd.kernels import native_moe, route, routed_moe, small_batch_moe
    from drama3_amd.mxfp4 import mxfp4_moe, quantize_experts_mxfp4

    fp8 = workloads.make_experts(torch.Generator("cpu").manual_seed(3), 16, 256, 128)
    experts = quantize_experts_mxfp4(fp8.to(device))
    assert (experts.num_experts, experts.hidden, experts.intermediate) == (16, 256, 128)

    def values(weight, inverse):
        w = f64(weight.float())
        w *= np.repeat(np.repeat(f64(inverse), 128, 1), 128, 2)
        return om.dequantize(*om.quantize(w.astype(np.float32).astype(np.float64)))

    v13, v2 = values(fp8.w13_weight, fp8.w13_scale_inv), values(fp8.w2_weight, fp8.w2_scale_inv)
    rng = np.random.default_rng(21)
    x = rows_of(rng, 30, 256).to(device)
    router = torch.from_numpy(rng.standard_normal((30, 16))).to(torch.bfloat16).to(device)
    weights, ids = route(router)
    out = mxfp4_moe(x, ids, weights, experts)
    within(out, *om.moe(f64(x), ids.cpu().numpy(), f64(weights), v13, v2))
    assert torch.equal(routed_moe(x, router, experts), out)
    assert torch.equal(small_batch_moe(x, ids, weights, experts), out)
    assert torch.equal(native_moe(x, ids, weights, experts, block_m=64), out)
    slots = torch.arange(30, device=device)
    padded = routed_moe(x, router, experts, row_slots=slots, padding_start=20)
    first = torch.where((slots >= 20)[:, None], ids[:1], ids), torch.where((slots >= 20)[:, None], weights[:1], weights)
    assert torch.equal(padded, mxfp4_moe(x, *first, experts))
    assert routed_moe(x[:0], router[:0], experts).shape == (0, 256)


def test_fp8_experts_without_checkpoint_rows_are_refused(device):
    from drama3_amd import workloads
    from drama3_amd.expert_weights import prepare_experts
    from drama3_amd.mxfp4 import quantize_experts_mxfp4

    fp8 = workloads.make_experts(torch.Generator("cpu").manual_seed(4), 2, 256, 128).to(device)
    want = quantize_experts_mxfp4(fp8)
    kept = quantize_experts_mxfp4(prepare_experts(fp8))
    assert torch.equal(kept.w13.codes, want.w13.codes) and torch.equal(kept.w2.scales, want.w2.scales)
    with pytest.raises(ValueError, match="fragment-major"):
        quantize_experts_mxfp4(prepare_experts(fp8, keep_reference=False))


def test_empty_batches(device):
    from drama3_amd import mxfp4 as mx

    rng = np.random.default_rng(22)
    packed, *_ = make_experts(rng, 4, 256, 128, device)
    codes, scales, _ = weight_of(rng, 4, 65, 256)
    weight = mx.prepare_mxfp4(codes.to(device), scales.to(device))
    one = mx.prepare_mxfp4(codes[0].to(device), scales[0].to(device))
    x = torch.empty((0, 256), dtype=torch.bfloat16, device=device)
    ids = torch.empty((0, 8), dtype=torch.int64, device=device)
    q, s = mx.quantize_mxfp4(x)
    assert q.shape == (0, 128) and s.shape == (0, 8)
    assert mx.dequantize_mxfp4(q, s).shape == (0, 256)
    assert mx.mxfp4_linear(x, one).shape == (0, 65)
    assert mx.grouped_mxfp4(x, torch.zeros(5, dtype=torch.int32, device=device), weight).shape == (0, 65)
    assert mx.mxfp4_moe(x, ids, ids.to(torch.bfloat16), packed).shape == (0, 256)


def test_refusals(device):
    from drama3_amd import mxfp4 as mx

    rng = np.random.default_rng(23)
    packed, *_ = make_experts(rng, 4, 256, 128, device)
    codes, scales, _ = (t.to(device) if torch.is_tensor(t) else t for t in weight_of(rng, 4, 64, 256))
    weight = mx.prepare_mxfp4(codes, scales)
    x = rows_of(rng, 6, 256).to(device)
    bounds = torch.tensor([0, 1, 2, 3, 6], dtype=torch.int32, device=device)
    ids = torch.zeros((6, 2), dtype=torch.int64, device=device)
    w = torch.ones((6, 2), device=device)

    def refused(kind, match, f, *args, **more):
        with pytest.raises(kind, match=match):
            f(*args, **more)

    refused(ValueError, "multiple of 32", mx.quantize_mxfp4, x[:, :40])
    refused(TypeError, "bfloat16", mx.quantize_mxfp4, x.half())
    refused(ValueError, "column stride", mx.quantize_mxfp4, x.T)
    refused(ValueError, "do not match", mx.dequantize_mxfp4, codes[0], scales[0][:, :4])
    refused(TypeError, "uint8", mx.dequantize_mxfp4, codes[0].to(torch.int32), scales[0])
    refused(TypeError, "float32", mx.dequantize_mxfp4, codes[0], scales[0], torch.float16)
    refused(ValueError, "multiple of 128", mx.prepare_mxfp4, codes[:, :, :48], scales[:, :, :3])
    refused(ValueError, "one matrix", mx.mxfp4_linear, x, weight)
    refused(TypeError, "bfloat16", mx.grouped_mxfp4, x.float(), bounds, weight)
    refused(ValueError, "K=256", mx.grouped_mxfp4, x[:, :128], bounds, weight)
    refused(TypeError, "int32", mx.grouped_mxfp4, x, bounds.long(), weight)
    refused(ValueError, "one more than", mx.grouped_mxfp4, x, bounds[:4], weight)
    refused(ValueError, "out must be", mx.grouped_mxfp4, x, bounds, weight, out=x)
    refused(TypeError, "out must be", mx.grouped_mxfp4, x, bounds, weight, out=x[:, :64].float())
    refused(ValueError, "prepare_mxfp4", mx.grouped_mxfp4, x, bounds, packed.w13)
    refused(ValueError, "multiples of 128", mx.prepare_mxfp4_experts, codes, scales, codes, scales)
    refused(TypeError, "int32 or int64", mx.mxfp4_moe, x, ids.to(torch.int16), w, packed)
    refused(TypeError, "bfloat16 or float32", mx.mxfp4_moe, x, ids, w.half(), packed)
    refused(ValueError, "T rows", mx.mxfp4_moe, x, ids[:5], w[:5], packed)
    refused(ValueError, "hidden size 256", mx.mxfp4_moe, x[:, :128], ids, w, packed)
    refused(ValueError, "top_k 17", mx.mxfp4_moe, x, ids[:, :1].expand(6, 17), w[:, :1].expand(6, 17), packed)
    buffer = torch.zeros((6, 400), dtype=torch.bfloat16, device=device)
    refused(ValueError, "overlap", mx.grouped_mxfp4, buffer[:, :256], bounds, weight, out=buffer[:, 200:264])
    mx.grouped_mxfp4(buffer[:, :256], bounds, weight, out=buffer[:, 256:320])
    refused(ValueError, "prepare_mxfp4", mx.Mxfp4Weight, weight.codes, weight.scales, 5, 64, 256)
    refused(ValueError, "prepare_mxfp4", mx.Mxfp4Weight, weight.codes, weight.scales[8:], 4, 64, 256)
    refused(ValueError, "prepare_mxfp4_experts", mx.Mxfp4Experts, packed.w2, packed.w2)
    other, *_ = make_experts(rng, 4, 128, 128, device)
    refused(ValueError, "one device", mx.Mxfp4Experts, packed.w13, other.w2)
    # the refused calls left nothing behind
    assert torch.equal(mx.mxfp4_moe(x, ids, w, packed), mx.mxfp4_moe(x, ids, w, packed))


# ---------------------------------------------------------------------------
def test_together_captured_replayed_and_on_streams(device):
    """Projection, routing, routed experts and a grouped product in one
    captured step, two graphs replayed in turn with eager work between, each
    replay against the eager results for the same inputs; then eager calls on
    two streams at once."""
    from drama3_amd import mxfp4 as mx
    from drama3_amd.kernels import routed_moe

    rng = np.random.default_rng(24)
    packed, *_ = make_experts(rng, 16, 256, 128, device)
    pc, ps, _ = weight_of(rng, 16, 256)
    router_weight = mx.prepare_mxfp4(pc.to(device), ps.to(device))
    gc, gs, _ = weight_of(rng, 3, 100, 256)
    group_weight = mx.prepare_mxfp4(gc.to(device), gs.to(device))

    def step(x, bounds):
        router = mx.mxfp4_linear(x, router_weight)
        y = routed_moe(x, router, packed)
        return router, y, mx.grouped_mxfp4(y, bounds, group_weight)

    def inputs(rows):
        ends = sorted(rng.integers(0, rows + 1, 4).tolist())
        return rows_of(rng, rows, 256).to(device), torch.tensor(ends, dtype=torch.int32, device=device)

    captured = []
    for rows in (7, 150):
        held = inputs(rows)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step(*held)
        captured.append((rows, graph, held, results))
    for _ in range(4):
        for rows, graph, held, results in captured:
            new = inputs(rows)
            for to, value in zip(held, new):
                to.copy_(value)
            graph.replay()
            torch.cuda.synchronize()
            for got, want in zip(results, step(*new)):
                assert torch.equal(got, want)

    jobs = [inputs(rows) for rows in (90, 64, 3, 200)]
    want = [step(*job) for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    got = []
    for i, job in enumerate(jobs * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step(*job))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for a, b in zip(results, want[i % 4]):
            assert torch.equal(a, b)


def test_large_batches_captured_and_replayed(device):
    """The kernels of many rows in one graph: tiles, boundaries to items, the
    pairs grouped by chunks and by the route sort; replays with other inputs
    and eager work between, each against the eager results."""
    from drama3_amd import mxfp4 as mx

    rng = np.random.default_rng(26)
    packed, *_ = make_experts(rng, 24, 128, 128, device)
    lc, ls, _ = weight_of(rng, 1500, 128)
    linear = mx.prepare_mxfp4(lc.to(device), ls.to(device))
    gc, gs, _ = weight_of(rng, 5, 200, 128)
    groups = mx.prepare_mxfp4(gc.to(device), gs.to(device))

    def inputs():
        made = [rows_of(rng, 8300, 128).to(device)]
        ids, weights = make_routes(rng, 8300, 24, 8, 0.5)
        ids[rng.random(ids.shape) < 0.02] = -1
        ends = sorted(rng.integers(0, 8301, 6).tolist())
        return made + [ids.to(torch.int32).to(device), weights.to(torch.bfloat16).to(device),
                       torch.tensor(ends, dtype=torch.int32, device=device)]

    def step(x, ids, weights, bounds):
        return (mx.mxfp4_linear(x, linear), mx.grouped_mxfp4(x, bounds, groups), mx.mxfp4_moe(x, ids, weights, packed),
                mx.mxfp4_moe(x[:1500], ids[:1500], weights[:1500], packed),
                mx.mxfp4_moe(x[:700], ids[:700], weights[:700], packed))

    held = inputs()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*held)
    for _ in range(4):
        new = inputs()
        for to, value in zip(held, new):
            to.copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(results, step(*new)):
            assert torch.equal(got, want)


def test_calls_from_two_threads(device):
    """Two host threads, a stream each, the same weights."""
    import threading

    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(27)
    packed, *_ = make_experts(rng, 16, 256, 128, device)
    jobs = []
    for rows in (40, 500):
        ids, weights = make_routes(rng, rows, 16, 8)
        jobs.append((rows_of(rng, rows, 256).to(device), ids.to(device), weights.to(torch.bfloat16).to(device)))
    want = [mxfp4_moe(*job, packed) for job in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.device(device), torch.cuda.stream(torch.cuda.Stream(device)):
            for _ in range(20):
                got[i].append(mxfp4_moe(*jobs[i], packed))
            torch.cuda.current_stream(device).synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(out, want[i]) for out in got[i])


# ---------------------------------------------------------------------------
def moe_path(rows, top_k, experts, hidden, inter):
    """How a batch runs, told by its workspace: ``few`` keeps activations only,
    ``scan`` the ranks' rows too, ``sorted`` and ``tiled`` also the route list
    and its items, ``tiled`` the quantised rows besides."""
    from drama3_amd import _lib

    lib, pairs = _lib.load(), rows * top_k
    size = lib.d3_mxfp4_moe_workspace(rows, top_k, experts, hidden, inter)
    slack = 2048  # every array starts at a multiple of 256 bytes
    size -= pairs * -(-inter // 256) * 136
    if size <= slack:
        return "few"
    size -= 4 * pairs * hidden
    if size <= slack:
        return "scan"
    size -= 4 * pairs + 16 * lib.d3_max_items(pairs, experts, 16)
    return "sorted" if size <= slack else "tiled"


@pytest.mark.parametrize("path, rows, experts, hidden, inter", [
    ("few", 3, 4, 256, 128), ("scan", 600, 16, 256, 128), ("sorted", 600, 512, 256, 640),
    ("tiled", 1500, 8, 256, 128), ("tiled", 1300, 8, 384, 640), ("tiled", 1320, 8, 256, 1152)])
def test_moe_ranks_that_cancel_keep_fp32(device, path, rows, experts, hidden, inter):
    """Two ranks' results of 6144 and a little more, weighted 1 and -1: every
    product and sum is exact in fp32, so the difference has to be.  (In 16 bits
    they lie 4 apart.)"""
    from drama3_amd.mxfp4 import mxfp4_moe, prepare_mxfp4_experts

    assert moe_path(rows, 2, experts, hidden, inter) == path
    # act = silu(64 x) * (6 / 64) x = 6 x^2 in every column, x 1 or 2
    w13 = np.zeros((2, 2 * inter, hidden))
    w13[:, :inter, 0], w13[:, inter:, 0] = 64, 6 / 64
    w2 = np.zeros((2, hidden, inter))
    w2[:, :, 0] = 1024
    little = om.GRID[np.arange(hidden) % 8]
    w2[0, :, 40] = little
    which = (torch.arange(experts, device=device) > 0).long()  # expert 0, and copies of expert 1
    packed = prepare_mxfp4_experts(*(torch.from_numpy(t).to(device)[which] for w in (w13, w2) for t in om.quantize(w)))
    scale = np.where(np.arange(rows) % 3, 1.0, 2.0)
    x = torch.zeros((rows, hidden), dtype=torch.bfloat16)
    x[:, 0] = torch.from_numpy(scale)
    ids = torch.tensor([0, 1], dtype=torch.int32).expand(rows, 2).contiguous()
    weights = torch.tensor([1.0, -1.0]).expand(rows, 2).contiguous()
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    assert np.array_equal(f64(out), 6 * little * scale[:, None] ** 2)


def test_grouped_boundaries_that_do_not_ascend_stay_in_their_list(device):
    """Half of 65,536 groups claim every row, more work items together than 31
    bits count.  Which of them a row is multiplied by is not said; here all are
    the same, so the rows are known."""
    from drama3_amd.mxfp4 import grouped_mxfp4, mxfp4_linear, prepare_mxfp4

    rng = np.random.default_rng(29)
    rows, groups = (1 << 23) + 1000, 1 << 16
    x = rows_of(rng, 1, 128).to(device)
    codes, scales, _ = (t.to(device) if torch.is_tensor(t) else t for t in weight_of(rng, 1, 128))
    weight = prepare_mxfp4(codes.expand(groups, 1, 64), scales.expand(groups, 1, 4))
    bounds = torch.arange(groups + 1, dtype=torch.int32, device=device) % 2 * rows
    out = grouped_mxfp4(x.expand(rows, 128), bounds, weight, out=torch.zeros(rows, 1, dtype=torch.bfloat16, device=device))
    assert (out == mxfp4_linear(x, prepare_mxfp4(codes, scales))).all()


def test_sizes_past_32_bits_are_refused(device):
    """Sizes whose low 32 bits would be fine."""
    from drama3_amd import mxfp4 as mx

    def refused(match, f, *args):
        with pytest.raises(ValueError, match=match):
            f(*args)

    u8 = dict(dtype=torch.uint8, device=device)
    width = (1 << 32) + 128
    refused("below 2.31", mx.quantize_mxfp4, torch.empty((1, width), dtype=torch.bfloat16, device=device))
    codes, scales = torch.empty((1, width // 2), **u8), torch.empty((1, width // 32), **u8)
    refused("below 2.31", mx.dequantize_mxfp4, codes, scales)
    refused("below 2.31", mx.prepare_mxfp4, codes, scales)
    rng = np.random.default_rng(30)
    packed, *_ = make_experts(rng, 4, 256, 128, device)
    w2 = packed.w2
    refused("below 2.31", mx.Mxfp4Weight, w2.codes, w2.scales, 4 + (1 << 32), w2.n, w2.k)
    refused("below 2.31", mx.Mxfp4Weight, w2.codes, w2.scales, 4, w2.n, w2.k + (1 << 32))
    x = rows_of(rng, 1, 256).to(device)
    ids = torch.zeros((1, 1), dtype=torch.int32, device=device).expand(1, (1 << 32) + 8)
    refused("top_k 4294967304", mx.mxfp4_moe, x, ids, torch.ones((1, 1), device=device).expand(ids.shape), packed)


def test_routed_on_the_device_of_its_rows(device, monkeypatch):
    """Both launches before the experts run with the rows' device current, the
    reserved-padding router's too; a router of another device is refused."""
    from drama3_amd import kernels, moe_input

    rng = np.random.default_rng(31)
    packed, *_ = make_experts(rng, 16, 256, 128, device)
    x = rows_of(rng, 30, 256).to(device)
    router = torch.from_numpy(rng.standard_normal((30, 16))).to(torch.bfloat16).to(device)
    slots = torch.arange(30, device=device)
    want = kernels.routed_moe(x, router, packed, row_slots=slots, padding_start=20)
    current, seen = [], []
    real = torch.cuda.device

    class Recorded(real):
        def __enter__(self):
            current.append(self.idx)
            return super().__enter__()

        def __exit__(self, *what):
            current.pop()
            return super().__exit__(*what)

    monkeypatch.setattr(torch.cuda, "device", Recorded)
    for module in (kernels, moe_input):
        def recorded(name, *args, call=module.call):
            seen.append((name, current[-1:]))
            return call(name, *args)

        monkeypatch.setattr(module, "call", recorded)
    out = kernels.routed_moe(x, router, packed, row_slots=slots, padding_start=20)
    assert seen == [("d3_prepare_moe_input", [device.index]), ("d3_route", [device.index])]
    assert torch.equal(out, want)

    class Elsewhere(torch.Tensor):
        device = property(lambda self: torch.device("cuda:1"))

    with pytest.raises(ValueError, match="router is on cuda:1"):
        kernels.routed_moe(x, router.as_subclass(Elsewhere), packed)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bounds", [b + b[-1:] for b in GROUPS])
@pytest.mark.parametrize("k, n", [(128, 300), (384, 50), (640, 129), (1152, 1), (1152, 200)])
def test_grouped_walked(device, bounds, k, n):
    """The one launch that walks each group's row tiles itself (no workspace):
    one, two and four slices of the contraction, groups of one to four tiles,
    rows of no group zeroed or, in a given column slice, left alone."""
    from drama3_amd import _lib
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    assert _lib.load().d3_mxfp4_grouped_workspace(100, 7, 1, n, k) == 0
    rng = np.random.default_rng(sum(bounds) % 1000 + k + n)
    x = rows_of(rng, 100, k + 3)[:, 2:k + 2]
    codes, scales, values = weight_of(rng, 7, n, k)
    weight = prepare_mxfp4(codes.to(device), scales.to(device))
    boundaries = torch.tensor(bounds, dtype=torch.int32, device=device)
    want, bound, live = grouped_oracle(x, bounds, values)
    live = torch.from_numpy(live).to(device)
    out = grouped_mxfp4(x.to(device), boundaries, weight)
    within(out, want, bound)
    assert not out[~live].any()
    buffer = torch.full((200, n + 9), -3.0, dtype=torch.bfloat16, device=device)
    given = grouped_mxfp4(x.to(device), boundaries, weight, out=buffer[::2, 5:5 + n])
    assert torch.equal(given, torch.where(live[:, None], out, -3.0))
    assert (buffer[:, :5] == -3).all() and (buffer[:, 5 + n:] == -3).all() and (buffer[1::2] == -3).all()


@pytest.mark.parametrize("bounds", [[0, 48], [3, 40], [-7, 1000], [48, 48], [0, 0], [20, 37]])
@pytest.mark.parametrize("k", [256, 896])
def test_grouped_walked_by_one_group(device, bounds, k):
    from drama3_amd import _lib
    from drama3_amd.mxfp4 import grouped_mxfp4, prepare_mxfp4

    assert _lib.load().d3_mxfp4_grouped_workspace(48, 1, 1, 130, k) == 0
    rng = np.random.default_rng(32 + k)
    x = rows_of(rng, 48, k)
    codes, scales, values = weight_of(rng, 1, 130, k)
    out = grouped_mxfp4(x.to(device), torch.tensor(bounds, dtype=torch.int32, device=device),
                        prepare_mxfp4(codes.to(device), scales.to(device)))
    want, bound, live = grouped_oracle(x, bounds, values)
    within(out, want, bound)
    assert not out[~torch.from_numpy(live).to(device)].any()


def many_experts(rng, distinct, experts, hidden, inter, device):
    """``make_experts`` of which expert e is a copy of expert e % distinct, and
    the ids by which the oracle finds it among the distinct ones."""
    from drama3_amd.mxfp4 import prepare_mxfp4_experts

    c13, s13, v13 = weight_of(rng, distinct, 2 * inter, hidden)
    c2, s2, v2 = weight_of(rng, distinct, hidden, inter)
    which = torch.arange(experts, device=device) % distinct
    packed = prepare_mxfp4_experts(*(t.to(device)[which] for t in (c13, s13, c2, s2)))

    def found(ids):
        ids = ids.numpy().astype(np.int64)
        return np.where((ids >= 0) & (ids < experts), ids % distinct, -1)

    return packed, v13, v2, found


@pytest.mark.parametrize("rows, hidden, inter", [(40, 512, 1024), (40, 1152, 128), (50, 1152, 1024), (150, 512, 640),
                                                 (17, 256, 640)])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_moe_sorted_and_streamed(device, rows, hidden, inter, id_type):
    """Routes sorted into items of 16 rows and streamed, the path of a full
    decode bucket: one, two and four slices of either product, ids of no
    expert, an expert of every row."""
    from drama3_amd.mxfp4 import mxfp4_moe

    assert moe_path(rows, 8, 200, hidden, inter) == "sorted"
    rng = np.random.default_rng(rows + hidden + inter)
    packed, v13, v2, found = many_experts(rng, 7, 200, hidden, inter, device)
    x = rows_of(rng, rows, hidden + 5)[:, 3:hidden + 3]
    ids, weights = make_routes(rng, rows, 200, 8)
    ids[rng.random(ids.shape) < 0.1] = -1
    ids[1], ids[2, 5] = 200, 2 ** 31 - 1
    ids, weights = ids.to(id_type), weights.to(torch.bfloat16)
    for skewed in (False, True):
        if skewed:
            ids[:, 3], ids[5:, 0] = 190, 190  # (twice in a row)
        out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
        within(out, *om.moe(f64(x), found(ids), f64(weights), v13, v2))


@pytest.mark.parametrize("rows, experts, hidden, inter, top_k", [(5, 60, 384, 256, 11), (8, 16, 256, 640, 16),
                                                                 (1, 20, 128, 128, 9), (9, 512, 1152, 128, 13)])
def test_moe_of_few_pairs_and_many_ranks(device, rows, experts, hidden, inter, top_k):
    """More ranks than the down product's workgroup has waves."""
    from drama3_amd.mxfp4 import mxfp4_moe

    assert moe_path(rows, top_k, experts, hidden, inter) == "few"
    rng = np.random.default_rng(rows + top_k)
    packed, v13, v2, found = many_experts(rng, 5, experts, hidden, inter, device)
    x = rows_of(rng, rows, hidden)
    ids, weights = make_routes(rng, rows, experts, top_k)
    ids[0, 8], ids[rows - 1, 2] = experts, -1
    weights[0, 8] = float("nan")  # of a rank that adds nothing
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(torch.float32).to(device), packed)
    within(out, *om.moe(f64(x), found(ids), f64(weights.to(torch.float32)), v13, v2))


@pytest.mark.parametrize("rows, experts, top_k, id_type", [
    (1100, 512, 8, torch.int32), (4100, 3, 4, torch.int64), (9001, 1, 1, torch.int32),  # grouped by chunks
    (4500, 512, 16, torch.int64), (33000, 3, 2, torch.int32), (66001, 1, 1, torch.int64)])  # by the route sort
def test_moe_many_pairs_of_few_and_many_experts(device, rows, experts, top_k, id_type):
    from drama3_amd.mxfp4 import mxfp4_moe

    assert moe_path(rows, top_k, experts, 128, 128) == "tiled"
    rng = np.random.default_rng(rows)
    packed, v13, v2, found = many_experts(rng, 9, experts, 128, 128, device)
    x = rows_of(rng, rows, 128)
    ids = torch.from_numpy(rng.integers(0, experts, (rows, top_k)))
    ids[torch.from_numpy(rng.random((rows, top_k)) < 0.5)] = experts - 1  # half of them of one expert
    none = torch.from_numpy(rng.random((rows, top_k)) < 0.02)
    ids[none] = experts if id_type == torch.int32 else (1 << 32)  # (a low half that names one)
    ids, weights = ids.to(id_type), torch.from_numpy(rng.random((rows, top_k))).to(torch.float32)
    out = mxfp4_moe(x.to(device), ids.to(device), weights.to(device), packed)
    pick = np.concatenate([rng.choice(rows, 100, replace=False), np.flatnonzero(none.any(1))[:30], [0, rows - 1]])
    want, bound = om.moe(f64(x)[pick], found(ids)[pick], f64(weights)[pick], v13, v2)
    within(out[torch.from_numpy(pick).to(device)], want, bound)


@pytest.mark.parametrize("experts, hidden, inter, paths", [
    (200, 1152, 128, {1: "few", 16: "few", 40: "sorted", 190: "sorted", 260: "tiled"}),
    (16, 512, 256, {1: "few", 5: "few", 40: "scan", 150: "scan", 400: "tiled"})])
def test_batches_of_every_path_agree(device, experts, hidden, inter, paths):
    """The first rows of a batch alone and with others, one size a path.  What
    may differ is the order of the fp32 sums, and with it a code of an
    activation at a border: any two results lie within twice the bound that
    either has to the definition."""
    from drama3_amd.mxfp4 import mxfp4_moe

    rng = np.random.default_rng(33 + experts)
    packed, v13, v2, found = many_experts(rng, 6, experts, hidden, inter, device)
    most = max(paths)
    x = rows_of(rng, most, hidden)
    ids, weights = make_routes(rng, most, experts, 8)
    on = [t.to(device) for t in (x, ids, weights.to(torch.float32))]
    results = {}
    for rows, path in paths.items():
        assert moe_path(rows, 8, experts, hidden, inter) == path
        results[rows] = f64(mxfp4_moe(*(t[:rows] for t in on), packed))
    few = min(r for r in paths if r > 1)
    want, bound = om.moe(f64(x[:few]), found(ids[:few]), f64(on[2][:few]), v13, v2)
    for a in results.values():
        for b in results.values():
            n = min(len(a), len(b), few)
            assert (np.abs(a[:n] - b[:n]) <= 2 * bound[:n]).all()
