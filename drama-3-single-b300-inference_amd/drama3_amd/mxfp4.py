"""MXFP4 (OCP Microscaling, 4 bits): quantisation of rows, and the products of
quantised rows with MXFP4 weights: one matrix, one per group of rows, and the
routed SwiGLU experts.  No counterpart in the reference, whose experts are FP8
in 128 x 128 blocks: MXFP4 experts take half their bytes, and gfx950 multiplies
them at twice the FP8 rate.

A row of K elements is ``K / 2`` bytes of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4,
6, bit 3 the sign; the even element in the low nibble) and ``K / 32`` e8m0
scales, one byte per 32 elements: ``2 ** (code - 127)``, 255 = NaN.  A block's
scale is ``2 ** (floor(log2(amax)) - 2)`` (at least 2 ** -127), its elements
``e2m1(x / scale)``, ties to the even code, magnitudes above 6 to 6; a block
that holds an infinity or a NaN reads as NaN throughout.

Weights are packed once (``prepare_mxfp4``, ``prepare_mxfp4_experts``); every
product takes bf16 rows and quantises them itself, to the same codes in a batch
of any size; codes times codes are summed in fp32 and rounded to bf16 once.  The
order of a sum does depend on the batch (how a product runs follows from its
sizes), so a row's results may differ in their last bit, and those of the routed
experts by what an activation on a border between two codes adds.  The same call
gives the same bits.

Every call allocates what it returns and its workspace from torch's allocator
on the current stream: calls on different streams share nothing, and a
captured graph keeps its own workspace.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import ptr
from .pipeline import require_cuda

BLOCK = 32  # elements per scale
ORDER_ROWS, ORDER_GATE_UP = 0, 1  # row order of a packed weight
_FLOAT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_INT = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}
_MOST = (1 << 31) - 1  # of an int32 argument: ctypes cuts more off without a word


# Where rows are few, what a call costs the host counts (6.5 us with one launch,
# 3.4 of them the launch): sizes are given to torch.empty one by one (1.0 us; as
# a tuple 1.35), a tensor's length is taken from its shape (len: 0.27), and the
# current stream's handle without building a torch.cuda.Stream (1.7).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is None:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


@functools.cache
def _entry(name: str):
    return getattr(_lib.load(), name)


def _call(device: torch.device, name: str, *args) -> None:
    """``_lib.call`` with the current stream of ``device`` appended, launched
    with ``device`` current (a stream takes kernels of its own device only)."""
    index = device.index
    if index == torch.cuda.current_device():
        status = _entry(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = _entry(name)(*args, _raw_stream(index))
    if status:
        _lib.fail(status)


def _same_device(x: torch.Tensor, t: torch.Tensor, name: str) -> None:
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, the rows on {x.device}")


def _workspace(size: int, x: torch.Tensor):
    """(the tensor to hold on to, its address) of a call's workspace; sizes
    below 1 need none, or are refused by the call itself."""
    if size <= 0:
        return None, None
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    return workspace, workspace.data_ptr()


def _check_rows(x: torch.Tensor, dtypes=(torch.bfloat16,)) -> None:
    require_cuda(x)
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError("x must be 2-D with unit column stride")
    if x.dtype not in dtypes:
        raise TypeError("x must be " + " or ".join(str(d).removeprefix("torch.") for d in dtypes))


def _check_codes(codes: torch.Tensor, scales: torch.Tensor) -> None:
    require_cuda(codes, scales)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("codes and scales must be uint8")
    if (codes.dim() != scales.dim() or codes.shape[:-1] != scales.shape[:-1]
            or codes.shape[-1] * 2 != scales.shape[-1] * BLOCK):
        raise ValueError("codes [..., K / 2] and scales [..., K / 32] do not match")
    _same_device(codes, scales, "scales")


def quantize_mxfp4(x: torch.Tensor):
    """bf16 or f32 rows [T, K] (K a multiple of 32, any row stride) ->
    ``(codes uint8 [T, K / 2], scales uint8 [T, K / 32])``."""
    _check_rows(x, _FLOAT)
    rows, width = x.shape
    if width == 0 or width % BLOCK or width > _MOST:
        raise ValueError(f"row width {width} must be a multiple of {BLOCK} below 2^31")
    codes = torch.empty(rows, width // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, width // BLOCK, dtype=torch.uint8, device=x.device)
    _call(x.device, "d3_mxfp4_quantize", ptr(x), _FLOAT[x.dtype], x.stride(0), rows, width,
          ptr(codes), ptr(scales))
    return codes, scales


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values MXFP4 rows stand for: bf16 (exact) or f32 [T, K]."""
    _check_codes(codes, scales)
    if codes.dim() != 2 or codes.shape[1] == 0:
        raise ValueError("codes must be [T, K / 2]")
    if dtype not in _FLOAT:
        raise TypeError("dtype must be bfloat16 or float32")
    codes, scales = codes.contiguous(), scales.contiguous()
    rows, half = codes.shape
    width = 2 * half
    if width > _MOST:
        raise ValueError(f"row width {width} must be below 2^31")
    out = torch.empty(rows, width, dtype=dtype, device=codes.device)
    _call(codes.device, "d3_mxfp4_dequantize", ptr(codes), ptr(scales), rows, width, ptr(out),
          _FLOAT[dtype])
    return out


@dataclass(frozen=True)
class Mxfp4Weight:
    """Packed MXFP4 weights of one product: ``experts`` matrices [N, K]
    (``prepare_mxfp4``); ``codes`` / ``scales`` are in the kernels' layout."""

    codes: torch.Tensor
    scales: torch.Tensor
    experts: int
    n: int
    k: int
    order: int = ORDER_ROWS

    def __post_init__(self):
        """The kernels take the sizes as given: they have to be the buffers'."""
        require_cuda(self.codes, self.scales)
        _same_device(self.codes, self.scales, "scales")
        if max(self.experts, self.n, self.k) > _MOST:
            raise ValueError(f"packed weights of [{self.experts}, {self.n}, {self.k}]: each must be below 2^31")
        for t, scales in ((self.codes, 0), (self.scales, 1)):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != _entry("d3_mxfp4_packed_bytes")(
                    self.experts, self.n, self.k, scales):
                raise ValueError("packed codes and scales do not hold [experts, n, k]; make them with prepare_mxfp4")

    @property
    def device(self) -> torch.device:
        return self.codes.device


@dataclass(frozen=True)
class Mxfp4Experts:
    """Routed SwiGLU experts on MXFP4 weights (``prepare_mxfp4_experts``)."""

    w13: Mxfp4Weight
    w2: Mxfp4Weight

    def __post_init__(self):
        w13, w2 = self.w13, self.w2
        if w13.order != ORDER_GATE_UP or w2.order != ORDER_ROWS:
            raise ValueError("experts must come from prepare_mxfp4_experts")
        if (w13.experts, w13.n, w13.k) != (w2.experts, 2 * w2.k, w2.n) or w13.device != w2.device:
            raise ValueError("expert weights must be w13 [E, 2I, H], w2 [E, H, I] on one device")

    @property
    def num_experts(self) -> int:
        return self.w13.experts

    @property
    def hidden(self) -> int:
        return self.w13.k

    @property
    def intermediate(self) -> int:
        return self.w2.k


def _prepare(codes: torch.Tensor, scales: torch.Tensor, order: int) -> Mxfp4Weight:
    _check_codes(codes, scales)
    if codes.dim() == 2:
        codes, scales = codes[None], scales[None]
    if codes.dim() != 3 or 0 in codes.shape:
        raise ValueError("weights must be [N, K / 2] or [E, N, K / 2] codes")
    experts, n, k = codes.shape[0], codes.shape[1], 2 * codes.shape[2]
    if k % 128 or max(experts, n, k) > _MOST:
        raise ValueError(f"K={k} must be a multiple of 128, and it, N={n} and the experts below 2^31")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    size = _entry("d3_mxfp4_packed_bytes")
    u8 = dict(dtype=torch.uint8, device=codes.device)
    packed = torch.empty(size(experts, n, k, 0), **u8)
    packed_scales = torch.empty(size(experts, n, k, 1), **u8)
    _call(codes.device, "d3_mxfp4_pack", ptr(codes), ptr(scales), experts, n, k, order, ptr(packed),
          ptr(packed_scales))
    return Mxfp4Weight(packed, packed_scales, experts, n, k, order)


def prepare_mxfp4(codes: torch.Tensor, scales: torch.Tensor) -> Mxfp4Weight:
    """Weights [N, K] or [E, N, K] as ``quantize_mxfp4`` gives them (K a
    multiple of 128, any N) -> the packed weight of ``mxfp4_linear`` /
    ``grouped_mxfp4``.  The arguments are not needed afterwards."""
    return _prepare(codes, scales, ORDER_ROWS)


def prepare_mxfp4_experts(w13_codes, w13_scales, w2_codes, w2_scales) -> Mxfp4Experts:
    """``w13`` [E, 2I, H] (rows [gate; up]) and ``w2`` [E, H, I] as codes and
    scales (H and I multiples of 128) -> the experts of ``mxfp4_moe``."""
    if w13_codes.dim() != 3 or w2_codes.dim() != 3:
        raise ValueError("expert weights must be [E, N, K / 2] codes")
    experts, two_i, half_h = w13_codes.shape
    if w2_codes.shape != (experts, 2 * half_h, two_i // 4) or two_i % 256 or half_h % 64:
        raise ValueError("expert weights must be w13 [E, 2I, H], w2 [E, H, I], H and I multiples of 128")
    _same_device(w13_codes, w2_codes, "w2_codes")
    return Mxfp4Experts(_prepare(w13_codes, w13_scales, ORDER_GATE_UP),
                        _prepare(w2_codes, w2_scales, ORDER_ROWS))


def quantize_experts_mxfp4(experts) -> Mxfp4Experts:
    """FP8 block-scaled experts (``w13_weight``, ``w13_scale_inv``,
    ``w2_weight``, ``w2_scale_inv``: the MoE operators' contract) rounded to
    MXFP4, one expert at a time, at load time.  They have to hold checkpoint
    rows: not after ``prepare_experts(..., keep_reference=False)``."""
    if any(getattr(experts, f"d3_{name}_fragment_only", False) for name in ("w13", "w2")):
        raise ValueError("experts hold only fragment-major codes; quantise them before "
                         "prepare_experts(keep_reference=False)")
    packed = []
    for weight, inverse, order in ((experts.w13_weight, experts.w13_scale_inv, ORDER_GATE_UP),
                                   (experts.w2_weight, experts.w2_scale_inv, ORDER_ROWS)):
        require_cuda(weight, inverse)
        if weight.dim() != 3 or weight.dtype != torch.float8_e4m3fn:
            raise TypeError("expert weights must be float8_e4m3fn [E, N, K]")
        e, n, k = weight.shape
        if n % 128 or k % 128 or inverse.shape != (e, n // 128, k // 128):
            raise ValueError("expert weights do not follow the 128x128 block layout")
        codes = torch.empty((e, n, k // 2), dtype=torch.uint8, device=weight.device)
        scales = torch.empty((e, n, k // BLOCK), dtype=torch.uint8, device=weight.device)
        for i in range(e):
            blocks = weight[i].float().view(n // 128, 128, k // 128, 128)
            values = (blocks * inverse[i].float()[:, None, :, None]).view(n, k)
            codes[i], scales[i] = quantize_mxfp4(values)
        packed.append(_prepare(codes, scales, order))
    return Mxfp4Experts(*packed)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether 2-D bf16 tensors of unit column stride may share an element:
    their spans meet, and they are not different columns of rows of one stride."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    apart = (b.data_ptr() - a.data_ptr()) // 2
    if apart >= (len(a) - 1) * a.stride(0) + a.shape[1]:
        return False
    stride = a.stride(0)
    if stride != b.stride(0) or stride == 0:
        return True
    return apart % stride < a.shape[1] or apart % stride + b.shape[1] > stride


def _product(x, boundaries, weight: Mxfp4Weight, out, zero_rest: bool) -> torch.Tensor:
    _check_rows(x)
    if weight.order != ORDER_ROWS:
        raise ValueError("weight holds gate and up rows; pack it with prepare_mxfp4")
    rows, k = x.shape
    if k != weight.k:
        raise ValueError(f"rows of width {k}, weight of K={weight.k}")
    _same_device(x, weight.codes, "weight")
    if out is None:
        out = torch.empty(rows, weight.n, dtype=torch.bfloat16, device=x.device)
    size = _entry("d3_mxfp4_grouped_workspace")(rows, weight.experts, boundaries is not None,
                                                  weight.n, k)
    workspace, at = _workspace(size, x)
    _call(x.device, "d3_mxfp4_grouped", ptr(x), x.stride(0), rows, ptr(boundaries), weight.experts,
          ptr(weight.codes), ptr(weight.scales), weight.n, k, ptr(out), out.stride(0),
          zero_rest, at, size)
    return out


def mxfp4_linear(x: torch.Tensor, weight: Mxfp4Weight) -> torch.Tensor:
    """``x`` bf16 [T, K], quantised to MXFP4, times the weight [N, K]
    transposed -> bf16 [T, N]."""
    if weight.experts != 1:
        raise ValueError(f"mxfp4_linear takes one matrix, the weight holds {weight.experts}")
    return _product(x, None, weight, None, False)


def grouped_mxfp4(x: torch.Tensor, boundaries: torch.Tensor, weight: Mxfp4Weight,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows ``[boundaries[e], boundaries[e + 1])`` of ``x`` bf16 [T, K],
    quantised to MXFP4, times matrix e of ``weight`` [E, N, K] transposed ->
    bf16 [T, N].

    ``boundaries`` int32 [E + 1], ascending, on the device (groups may be
    empty; values are clamped to [0, T]).  Rows of no group are zeros, or left
    as they were in a given ``out`` (bf16 [T, N], unit column stride, apart from
    ``x``)."""
    _check_rows(x)
    require_cuda(boundaries, out)
    if boundaries.dtype != torch.int32:
        raise TypeError("boundaries must be int32")
    if boundaries.shape != (weight.experts + 1,) or boundaries.stride(0) != 1:
        raise ValueError(f"boundaries must be contiguous [{weight.experts + 1}], one more than the experts")
    _same_device(x, boundaries, "boundaries")
    if out is not None:
        rows = x.shape[0]
        if out.dtype != torch.bfloat16:
            raise TypeError("out must be bfloat16")
        if out.shape != (rows, weight.n) or (weight.n > 1 and out.stride(1) != 1) or (
                rows > 1 and out.stride(0) < weight.n):
            raise ValueError(f"out must be [{rows}, {weight.n}] with unit column stride")
        _same_device(x, out, "out")
        if _overlap(x, out):
            raise ValueError("out must not overlap x")
    return _product(x, boundaries, weight, out, out is None)


def mxfp4_moe(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
              experts: Mxfp4Experts) -> torch.Tensor:
    """Routed SwiGLU experts: for row t and rank r with expert e =
    ``topk_ids[t, r]``, ``a = silu(G_e x) * (U_e x)`` and ``out[t] = sum_r
    topk_weights[t, r] * W2_e a`` in rank order, with x and a quantised to
    MXFP4 and fp32 sums (the ranks' rows too), rounded to bf16 [T, H] once.

    ``topk_ids`` int32 / int64 [T, k], k <= 16 (an id that names no expert
    adds nothing), ``topk_weights`` bf16 / f32 of the same shape."""
    _check_rows(x)
    require_cuda(topk_ids, topk_weights)
    if topk_ids.dim() != 2 or topk_ids.shape != topk_weights.shape or topk_ids.shape[0] != x.shape[0]:
        raise ValueError("topk_ids / topk_weights must be [T, k] for the T rows of x")
    if topk_ids.shape[1] > _MOST:
        raise ValueError(f"top_k {topk_ids.shape[1]} (1 to 16)")
    if topk_ids.dtype not in _INT:
        raise TypeError("topk_ids must be int32 or int64")
    if topk_weights.dtype not in _FLOAT:
        raise TypeError("topk_weights must be bfloat16 or float32")
    if x.shape[1] != experts.hidden:
        raise ValueError(f"rows of width {x.shape[1]}, experts of hidden size {experts.hidden}")
    ids, weights = topk_ids.contiguous(), topk_weights.contiguous()
    w13, w2 = experts.w13, experts.w2
    _same_device(x, ids, "topk_ids")
    _same_device(x, weights, "topk_weights")
    _same_device(x, w13.codes, "experts")
    rows, top_k = ids.shape
    out = torch.empty(rows, experts.hidden, dtype=torch.bfloat16, device=x.device)
    size = _entry("d3_mxfp4_moe_workspace")(rows, top_k, w13.experts, w13.k, w2.k)
    workspace, at = _workspace(size, x)
    _call(x.device, "d3_mxfp4_moe", ptr(x), x.stride(0), rows, ptr(ids), _INT[ids.dtype],
          ptr(weights), _FLOAT[weights.dtype], top_k, ptr(w13.codes), ptr(w13.scales),
          ptr(w2.codes), ptr(w2.scales), w13.experts, w13.k, w2.k, ptr(out), at, size)
    return out
