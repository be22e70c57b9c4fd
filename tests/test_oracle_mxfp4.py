"""The MXFP4 oracle against the format's definition, and what the operators
refuse before any launch (CPU only)."""

import numpy as np
import pytest
import torch

from oracle import mxfp4 as om


def test_codes_round_to_nearest_even_and_saturate():
    # one block whose maximum is in [4, 8): scale 1, every border and its neighbours
    v = np.zeros(32)
    v[:16] = [0.25, 0.2500001, 0.75, 0.7499999, 1.25, 1.2500001, 1.75, 1.7499999,
              2.5, 2.5000001, 3.5, 3.4999999, 5.0, 5.0000001, 7.9, 6.0]
    codes, scales = om.quantize(v[None])
    assert scales.tolist() == [[127]]
    want = [0, .5, 1, .5, 1, 1.5, 2, 1.5, 2, 3, 4, 3, 4, 6, 6, 6]
    assert om.dequantize(codes, scales)[0, :16].tolist() == want
    codes, scales = om.quantize(-v[None])
    assert om.dequantize(codes, scales)[0, :16].tolist() == [-x for x in want]


@pytest.mark.parametrize("amax, code", [(0.0, 0), (4.0, 127), (7.99, 127), (8.0, 128), (1.0, 125),
                                        (2.0 ** -126, 0), (2.0 ** -140, 0), (2.0 ** -124, 1),
                                        (float(np.finfo(np.float32).max), 252), (np.inf, 255),
                                        (np.nan, 255)])
def test_scale_codes(amax, code):
    x = np.zeros((1, 32))
    x[0, 7] = amax
    codes, scales = om.quantize(x)
    assert scales.tolist() == [[code]]
    values = om.dequantize(codes, scales)
    assert np.isnan(values).all() if code == 255 else np.isfinite(values).all()


def test_every_value_is_a_fixed_point():
    nibble = np.arange(16, dtype=np.uint8)
    codes = np.tile(np.stack([nibble | (nibble[::-1] << 4)]).ravel(), 1)[None]
    for scale in (1, 100, 127, 200, 250):
        scales = np.array([[scale]], dtype=np.uint8)
        again, same = om.quantize(om.dequantize(codes, scales))
        assert same.tolist() == scales.tolist() and np.array_equal(
            om.dequantize(again, same), om.dequantize(codes, scales))


def test_requantize_bounds_what_errors_can_do():
    rng = np.random.default_rng(5)
    v = rng.standard_normal((20, 64)) * np.exp(rng.standard_normal((20, 1)))
    error = np.full_like(v, 2e-3)
    best, worst = om.requantize(v, error)
    assert np.array_equal(best, om.dequantize(*om.quantize(v)))
    assert 0 < (worst > 0).mean() < 0.2
    for _ in range(20):
        moved = om.dequantize(*om.quantize(v + error * rng.uniform(-1, 1, v.shape)))
        assert (np.abs(moved - best) <= worst).all()


@pytest.fixture(scope="module")
def lib():
    from drama3_amd import _lib

    if not _lib.LIBRARY.exists():
        pytest.skip("library not built")
    return _lib


def test_c_entries_refuse_before_launching(lib):
    call = lib.call
    with pytest.raises(ValueError, match="multiple of 32"):
        call("d3_mxfp4_quantize", 16, 0, 48, 4, 48, 16, 16, None)
    with pytest.raises(ValueError, match="bf16 or f32"):
        call("d3_mxfp4_quantize", 16, 2, 64, 4, 64, 16, 16, None)
    with pytest.raises(ValueError, match="null"):
        call("d3_mxfp4_quantize", None, 0, 64, 4, 64, 16, 16, None)
    with pytest.raises(ValueError, match="alignment"):
        call("d3_mxfp4_quantize", 17, 0, 64, 4, 64, 16, 16, None)
    with pytest.raises(ValueError, match="16-byte"):
        call("d3_mxfp4_dequantize", 16, 16, 4, 64, 8, 0, None)
    with pytest.raises(ValueError, match="multiple of 128"):
        call("d3_mxfp4_pack", 16, 16, 1, 64, 192, 0, 16, 16, None)
    with pytest.raises(ValueError, match="multiple of 64"):
        call("d3_mxfp4_pack", 16, 16, 1, 96, 256, 1, 16, 16, None)
    with pytest.raises(ValueError, match="order"):
        call("d3_mxfp4_pack", 16, 16, 1, 64, 256, 2, 16, 16, None)
    grouped = [16, 256, 40, 16, 4, 16, 16, 64, 256, 16, 64, 0, 16, 1 << 30, None]

    def refused(match, entry, args, **changes):
        args = list(args)
        for at, value in changes.items():
            args[int(at[1:])] = value
        with pytest.raises(ValueError, match=match):
            call(entry, *args)

    refused("multiple of 128", "d3_mxfp4_grouped", grouped, a8=64)
    refused("need boundaries", "d3_mxfp4_grouped", grouped, a3=None)
    refused("null", "d3_mxfp4_grouped", grouped, a0=None)
    refused("row strides", "d3_mxfp4_grouped", grouped, a10=63)
    refused("alignment", "d3_mxfp4_grouped", grouped, a5=24)
    refused("workspace of 100", "d3_mxfp4_grouped", grouped, a2=4000, a13=100)
    refused("workspace of", "d3_mxfp4_grouped", grouped, a2=4000, a12=None)
    refused("experts 0", "d3_mxfp4_grouped", grouped, a4=0)
    refused("rows -1", "d3_mxfp4_grouped", grouped, a2=-1)
    moe = [16, 256, 40, 16, 3, 16, 0, 8, 16, 16, 16, 16, 16, 256, 128, 16, 16, 1 << 30, None]
    refused("multiples of 128", "d3_mxfp4_moe", moe, a14=64)
    refused("top_k 17", "d3_mxfp4_moe", moe, a7=17)
    refused("experts 513", "d3_mxfp4_moe", moe, a12=513)
    refused("int32 or int64", "d3_mxfp4_moe", moe, a4=0)
    refused("bf16 or f32", "d3_mxfp4_moe", moe, a6=2)
    refused("null", "d3_mxfp4_moe", moe, a3=None)
    refused("alignment", "d3_mxfp4_moe", moe, a10=20)
    refused("workspace of 64", "d3_mxfp4_moe", moe, a17=64)
    refused("pairs", "d3_mxfp4_moe", moe, a2=1 << 24)
    lib_ = lib.load()
    assert lib_.d3_mxfp4_moe_workspace(4, 8, 513, 256, 128) == -1
    assert lib_.d3_mxfp4_grouped_workspace(4, 8, 1, 64, 100) == -1
    assert lib_.d3_mxfp4_packed_bytes(0, 64, 256, 0) == -1
    # padded to whole row groups of 64 and steps of 256
    assert lib_.d3_mxfp4_packed_bytes(3, 65, 384, 0) == 3 * 128 * 512 // 2
    assert lib_.d3_mxfp4_packed_bytes(3, 65, 384, 1) == 3 * 128 * 512 // 32


def test_sizes_past_the_kernels_offsets_are_refused(lib):
    """Widths past the 32-bit views and launches of more threads than a grid
    holds: an error before anything is launched, whatever the pointers."""
    call, lib_ = lib.call, lib.load()
    huge = 1 << 62
    with pytest.raises(ValueError, match="2.36 elements"):
        call("d3_mxfp4_quantize", 16, 0, 0, (1 << 31) + 1, 32, 16, 16, None)
    with pytest.raises(ValueError, match="2.36 elements"):
        call("d3_mxfp4_dequantize", 16, 16, (1 << 31) + 1, 32, 16, 0, None)
    for rows, n, k, match in ((4, 64, (1 << 20) + 128, "K=1048704"), (4, (1 << 24) + 1, 128, "N=16777217"),
                              (1 << 30, 64, 128, "rows 1073741824"), ((1 << 30) - 1, 1 << 10, 128, "workgroups")):
        with pytest.raises(ValueError, match=match):
            call("d3_mxfp4_grouped", 16, k, rows, None, 1, 16, 16, n, k, 16, n, 0, 16, huge, None)
    with pytest.raises(ValueError, match="workgroups"):  # groups walked by their own workgroups
        call("d3_mxfp4_grouped", 16, 128, 1, 16, 1 << 16, 16, 16, 1 << 15, 128, 16, 1 << 15, 0, None, 0, None)

    def moe(rows, top_k, hidden, inter):
        call("d3_mxfp4_moe", 16, hidden, rows, 16, 3, 16, 0, top_k, 16, 16, 16, 16, 16, hidden, inter, 16, 16,
             huge, None)

    for args, match in (((4, 8, (1 << 20) + 128, 128), "hidden 1048704"), ((4, 8, 128, (1 << 20) + 128), "2.20"),
                        (((1 << 23) + 1, 8, 128, 128), "pairs"), ((1 << 62, 8, 128, 128), "pairs"),
                        ((1 << 24, 1, 128, 128), "workgroups"), ((1 << 23, 1, 1024, 128), "4 GiB")):
        with pytest.raises(ValueError, match=match):
            moe(*args)
    assert lib_.d3_mxfp4_grouped_workspace(4, 8, 1, 64, (1 << 20) + 128) == -1
    assert lib_.d3_mxfp4_moe_workspace(1 << 62, 8, 16, 256, 128) == -1


def test_empty_calls_need_no_buffers(lib):
    lib.call("d3_mxfp4_quantize", None, 0, 64, 0, 64, None, None, None)
    lib.call("d3_mxfp4_dequantize", None, None, 0, 64, None, 0, None)
    lib.call("d3_mxfp4_grouped", None, 256, 0, None, 1, None, None, 64, 256, None, 64, 0, None, 0, None)
    lib.call("d3_mxfp4_moe", None, 256, 0, None, 3, None, 0, 8, None, None, None, None, 16, 256, 128,
             None, None, 0, None)


def test_host_tensors_are_refused(lib):
    from drama3_amd import mxfp4 as mx

    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    codes, scales = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8)
    for made in (lambda: mx.quantize_mxfp4(x), lambda: mx.dequantize_mxfp4(codes, scales),
                 lambda: mx.prepare_mxfp4(codes, scales)):
        with pytest.raises(ValueError, match="device tensors"):
            made()
    with pytest.raises(ValueError, match="device tensors"):
        mx.Mxfp4Weight(codes, scales, 1, 2, 128)


def test_overlapping_rows_are_found():
    from drama3_amd.mxfp4 import _overlap

    flat = torch.zeros(4000, dtype=torch.bfloat16)
    wide = flat[:2000].view(20, 100)

    def shared(a, b):
        """By the elements themselves."""
        index = torch.arange(4000)
        at = [set(torch.as_strided(index, t.shape, t.stride(), t.storage_offset()).flatten().tolist()) for t in (a, b)]
        return bool(at[0] & at[1])

    views = [wide, wide[:, :60], wide[:, 60:], wide[:, 59:], wide[3:9, 20:60], wide[::2, :60], wide[5:6], wide[6:7],
             wide[5:6, 40:90], wide[12:, :60], wide[:0], torch.as_strided(flat, (20, 60), (100, 1), 80),
             torch.as_strided(flat, (20, 30), (0, 1), 70), flat[2000:].view(20, 100)]
    for a in views:
        for b in views:
            assert _overlap(a, b) == _overlap(b, a)
            assert _overlap(a, b) or not shared(a, b)
    assert not _overlap(wide[:, :60], wide[:, 60:]) and not _overlap(wide, flat[2000:].view(20, 100))
    assert not _overlap(wide[5:6], wide[6:7]) and not _overlap(wide[:0], wide)


def test_rows_of_more_threads_than_a_grid_are_refused(lib):
    """Their quantisation is a launch of its own, whose size their products' does not bound."""
    huge = 1 << 62
    for boundaries, experts in ((None, 1), (16, 8)):
        with pytest.raises(ValueError, match="2.37 elements"):
            lib.call("d3_mxfp4_grouped", 16, 0, 1 << 25, boundaries, experts, 16, 16, 1, 4096, 16, 1, 0, 16, huge, None)


def test_steps_of_fp8_experts_refuse_mxfp4_ones():
    """The decode, mixed and layer steps read their experts through these."""
    from drama3_amd.expert_weights import fc1_operands, fc2_operands, prepare_experts
    from drama3_amd.mxfp4 import Mxfp4Experts

    experts = object.__new__(Mxfp4Experts)
    for step in (fc1_operands, fc2_operands, prepare_experts):
        with pytest.raises(TypeError, match="FP8 weights .* not Mxfp4Experts"):
            step(experts)
