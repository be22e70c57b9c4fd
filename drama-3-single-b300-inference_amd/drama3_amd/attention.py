"""Attention over packed rows and a paged cache: rotary positions, appending keys
and values to the cache with the rotation on the way, and the attention of new
tokens over the cached ones, single ones and chunks alike.

What precedes the MoE step in the reference's attention layers
(``src/drama3/model.py:55-141``: rotary positions, paged decode over 16-token
pages, packed prefill), over the same packed rows and persistent slots.  The
reference calls libraries here: the semantics are this module's own.

A step of one layer, eager or captured::

    q = append_paged(cache, k, v, positions, row_slots, rope=rope, q=q)
    out = paged_attention(q, cache, layout, lengths)

``positions`` are tokens of a slot, what it holds already counted:
``runtime_state.DeviceRequests.load`` gives a single token's.
``packed_prefill.packed_row_metadata`` counts every sequence's rows from 0, which
is a whole prompt's, and gives rows behind the last boundary to the last sequence.
Chunks on top of cached tokens, and batches with such rows (boundaries from 0 to
``rows``), take from it::

    packed_row_metadata(layout.boundaries, layout.sequence_slots, capacity, positions, row_slots)
    new = layout.boundaries.diff()
    positions[:rows] += torch.repeat_interleave(lengths - new, new, output_size=rows)
    row_slots[rows:] = -1

``lengths`` counts a sequence's tokens with the new ones.  Every call allocates
what it returns and its workspace from torch's allocator on the current stream:
calls on different streams share nothing, and a captured graph keeps its own
workspace.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass, field

import torch

from . import _lib
from ._lib import ptr
from .mxfp4 import _MOST, _entry, _raw_stream, _same_device
from .packed_prefill import PackedLayout
from .pipeline import require_cuda

HEAD_DIMS = (64, 128, 256)  # of paged_attention
SCALINGS = ("none", "linear", "base", "bands")
_FLOAT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_ROWS = {torch.bfloat16: _lib.DTYPE_BF16}
_CACHE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float8_e4m3fn: _lib.DTYPE_E4M3}
_INT = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class Rope:
    """Rotary positions (``prepare_rope``): ``turns`` fp64 [rotary_dim / 2] on
    the device, revolutions of each pair a position; ``magnitude`` multiplies
    what is rotated.  Pairs are columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
    where ``interleaved``."""

    turns: torch.Tensor
    interleaved: bool = False
    magnitude: float = 1.0
    _struct: _lib.RopeStruct = field(init=False, repr=False, compare=False)
    _ref: object = field(init=False, repr=False, compare=False)

    def __post_init__(self):
        require_cuda(self.turns)
        if self.turns.dtype != torch.float64:
            raise TypeError("turns must be float64")
        if self.turns.dim() != 1 or not 0 < len(self.turns) <= 512 or not self.turns.is_contiguous():
            raise ValueError("turns must be contiguous [rotary_dim / 2], at most 512")
        object.__setattr__(self, "_struct", _lib.RopeStruct(
            ptr(self.turns), 2 * len(self.turns), int(self.interleaved), self.magnitude))
        object.__setattr__(self, "_ref", ctypes.byref(self._struct))

    @property
    def rotary_dim(self) -> int:
        return 2 * len(self.turns)


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_length: int = 0, slow: float = 1.0, fast: float = 32.0) -> list[float]:
    """Radians a position of each of the ``rotary_dim / 2`` pairs:
    ``f_i = base ** (-2 i / rotary_dim)``, scaled for contexts ``factor`` times
    as long as the ``original_length`` a model was trained on:

    ``"linear"``  f / factor (positions are interpolated);
    ``"base"``    the base grows to ``base * factor ** (R / (R - 2))``, so that the
                  slowest pair turns as under "linear" and the fastest as before;
    ``"bands"``   pairs that turn ``fast`` times and more within the original
                  length stay, those that turn ``slow`` times and less are
                  interpolated, in between by the share (YaRN, arXiv 2309.00071).
                  Loaders that ramp over the pair's index instead have other
                  frequencies in between: ``Rope(turns)`` takes any."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary width {rotary_dim} must be even and positive")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} is none of {SCALINGS}")
    if base <= 0 or factor <= 0:
        raise ValueError("base and factor must be positive")
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        return [f / factor for f in frequencies]
    if scaling == "bands":
        if original_length <= 0 or not slow < fast:
            raise ValueError("bands need the original length, and slow < fast")
        for i, f in enumerate(frequencies):
            turns = original_length * f / (2 * math.pi)
            kept = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
            frequencies[i] = kept * f + (1.0 - kept) * f / factor
    return frequencies


def prepare_rope(rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none",
                 factor: float = 1.0, original_length: int = 0, slow: float = 1.0, fast: float = 32.0,
                 magnitude: float | None = None, device="cuda") -> Rope:
    """The rotary positions of a model, once at load time (``rope_frequencies``
    says what the scalings are).  ``magnitude`` defaults to 1, with ``"bands"``
    to ``0.1 ln(factor) + 1`` (above 1 only)."""
    frequencies = rope_frequencies(rotary_dim, base, scaling, factor, original_length, slow, fast)
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "bands" and factor > 1 else 1.0
    turns = torch.tensor([f / (2 * math.pi) for f in frequencies], dtype=torch.float64, device=device)
    return Rope(turns, interleaved, magnitude)


# What a call costs the host counts where its rows are few: each tensor's shape,
# strides and device number are asked for once (a torch.device costs 0.2 us, its
# number 0.05).
def _heads(x: torch.Tensor, name: str, dtypes=_ROWS):
    """(rows, heads, head_dim, row stride, head stride, device number) of [T, heads, head_dim]."""
    index = x.get_device()
    if index < 0:
        require_cuda(x)
    if x.dim() != 3:
        raise ValueError(f"{name} must be [T, heads, head_dim] with unit column stride")
    rows, heads, dim = x.shape
    row, head, unit = x.stride()
    if not heads or not dim or (unit != 1 and dim > 1):
        raise ValueError(f"{name} must be [T, heads, head_dim] with unit column stride")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be " + " or ".join(str(d).removeprefix("torch.") for d in dtypes))
    if heads > _MOST or dim > _MOST:
        raise ValueError(f"{name}: sizes must be below 2^31")
    return rows, heads, dim, row, head, index


def _indices(t: torch.Tensor, name: str, count: int, x: torch.Tensor, index: int) -> int:
    """The type code of int32 or int64 [count] on the rows' device."""
    code = _INT.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be int32 or int64")
    if t.dim() != 1 or t.shape[0] != count or (count > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous [{count}]")
    if t.get_device() != index:
        _elsewhere(x, t, name)
    return code


def _elsewhere(x: torch.Tensor, t: torch.Tensor, name: str) -> None:
    require_cuda(t)
    _same_device(x, t, name)


def _launch(index: int, name: str, *args) -> None:
    """``mxfp4._call`` by the device's number."""
    if index == torch.cuda.current_device():
        status = _entry(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = _entry(name)(*args, _raw_stream(index))
    if status:
        _lib.fail(status)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(sizes: tuple, rows: int, heads: int, count: int, longest: int) -> int:
    """Of ``paged_attention``, for a cache of the given sizes (arithmetic alone)."""
    dtype, kv_heads, head_dim, page_size, max_pages = sizes
    part = 1 << 20  # (any address and stride: they have no part in it)
    struct = _lib.PagedCacheStruct(part, part, dtype, kv_heads, head_dim, page_size, 1, 0, 0, 0, 0, 0, 0, part, 0, 1, max_pages)
    return _entry("d3_paged_attention_workspace")(ctypes.byref(struct), rows, heads, count, longest)


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and last byte address a tensor may touch, and one more."""
    if t.numel() == 0:
        return 0, 0
    size = t.element_size()
    low = sum(min(0, (n - 1) * s) for n, s in zip(t.shape, t.stride()))
    high = sum(max(0, (n - 1) * s) for n, s in zip(t.shape, t.stride()))
    return t.data_ptr() + low * size, t.data_ptr() + (high + 1) * size


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a1 <= b0 or b1 <= a0


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory: element by element where their strides are alike and each
    steps over what the smaller ones reach (views of one buffer), else by their spans."""
    if _apart(a, b):
        return False
    size = a.element_size()
    offset = b.data_ptr() - a.data_ptr()
    if a.dim() != b.dim() or b.element_size() != size or offset % size:
        return True
    dims = []
    for n, m, s, t in zip(a.shape, b.shape, a.stride(), b.stride()):
        if n > 1 and m > 1 and s != t:
            return True
        if n > 1 or m > 1:
            dims.append((s if n > 1 else t, n, m))
    dims.sort(reverse=True)
    a_reach = b_reach = 1
    for s, n, m in reversed(dims):
        if s < max(a_reach, b_reach):
            return True
        a_reach, b_reach = a_reach + (n - 1) * s, b_reach + (m - 1) * s

    def met(offset, level):  # differences of the indices from this dimension on that come to the offset
        if level == len(dims):
            return offset == 0
        s, n, m = dims[level]
        near = offset // s
        return any(-m < d < n and met(offset - d * s, level + 1) for d in (near, near + 1))

    return met(offset // size, 0)


def _check_out(out: torch.Tensor, x: torch.Tensor, name: str, in_place: bool) -> None:
    """``out`` of the rows' type and shape, each element its own, apart from ``x`` (or ``x`` itself)."""
    require_cuda(out)
    if out.dtype != x.dtype:
        raise TypeError(f"{name} must be {str(x.dtype).removeprefix('torch.')}")
    rows, heads, dim = x.shape
    if out.shape != x.shape or (dim > 1 and out.stride(2) != 1):
        raise ValueError(f"{name} must be {list(x.shape)} with unit column stride")
    _same_device(x, out, name)
    row, head = out.stride(0), out.stride(1)
    if rows and ((heads > 1 and head < dim) or (rows > 1 and row < (heads - 1) * (head if heads > 1 else 0) + dim)):
        raise ValueError(f"{name} must hold rows of heads one behind the other")
    if in_place and out.data_ptr() == x.data_ptr() and out.stride() == x.stride():
        return
    if not _apart(out, x):
        raise ValueError(f"{name} must not overlap the rows")


def apply_rope(x: torch.Tensor, positions: torch.Tensor, rope: Rope, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotates ``x`` bf16 or f32 [T, heads, head_dim] (any row and head stride) by
    its rows' ``positions`` (int32 or int64 [T], any value): the first
    ``rope.rotary_dim`` columns of every head, the others stay.  Angles are taken
    in 64 bits, one rounding.  ``out`` (the rows' shape and type) may be ``x``."""
    rows, heads, dim, row, head, index = _heads(x, "x", _FLOAT)
    code = _indices(positions, "positions", rows, x, index)
    if rope.turns.get_device() != index:
        _elsewhere(x, rope.turns, "rope")
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=x.dtype, device=x.device)
        out_row, out_head = heads * dim, dim
    else:
        _check_out(out, x, "out", True)
        out_row, out_head, _ = out.stride()
    _launch(index, "d3_rope_rows", x.data_ptr(), _FLOAT[x.dtype], row, head, rows, heads, dim, positions.data_ptr(), code,
            rope._ref, out.data_ptr(), out_row, out_head)
    return out


# ---------------------------------------------------------------------------
# The paged cache
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class PagedCache:
    """Keys and values of one layer in pages: ``keys`` / ``values``
    [pages, kv_heads, page_size, head_dim], bf16 or float8_e4m3fn (any page, head
    and token stride of whole 16 bytes: a [pages, page_size, kv_heads, head_dim]
    buffer goes in as its ``transpose(1, 2)``), and ``page_table`` int32 [slots,
    max_pages]: token t of a slot lies in page ``page_table[slot, t // page_size]``
    at token ``t % page_size``.  Entries outside [0, pages) are unmapped: nothing
    is written there, and nothing attends them.  page_size is a power of two.

    Keys and values share no memory (two parts of one buffer do not).
    e4m3 codes stand for code * scale of their head, ``k_scale`` / ``v_scale``
    f32 [kv_heads] (None: 1).  Two slots may share pages that neither appends to.

    The cache holds on to the tensors: what they hold may change at any time
    (the page table between two replays of a graph, too), where they lie may not."""

    keys: torch.Tensor
    values: torch.Tensor
    page_table: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None
    _struct: _lib.PagedCacheStruct = field(init=False, repr=False, compare=False)
    _ref: object = field(init=False, repr=False, compare=False)
    _sizes: tuple = field(init=False, repr=False, compare=False)
    _spans: tuple = field(init=False, repr=False, compare=False)

    def __post_init__(self):
        """The kernels take the sizes as given: they have to be the tensors'."""
        keys, values, table = self.keys, self.values, self.page_table
        require_cuda(keys, values, table, self.k_scale, self.v_scale)
        if keys.dtype not in _CACHE or values.dtype != keys.dtype:
            raise TypeError("keys and values must both be bfloat16 or float8_e4m3fn")
        if keys.dim() != 4 or keys.shape != values.shape or 0 in keys.shape:
            raise ValueError("keys and values must be [pages, kv_heads, page_size, head_dim] of one shape")
        pages, kv_heads, page_size, head_dim = keys.shape
        if page_size & (page_size - 1):
            raise ValueError(f"page size {page_size} must be a power of two")
        if table.dtype != torch.int32:
            raise TypeError("page_table must be int32")
        if table.dim() != 2 or 0 in table.shape or (table.shape[1] > 1 and table.stride(1) != 1) or (
                table.shape[0] > 1 and table.stride(0) < table.shape[1]):
            raise ValueError("page_table must be [slots, max_pages] with unit column stride")
        if max(pages, kv_heads, head_dim, table.shape[0]) > _MOST or table.shape[1] * page_size > 1 << 30:
            raise ValueError("pages, heads and slots must be below 2^31, a slot's tokens at most 2^30")
        part = 16 // keys.element_size()
        for t, name in ((keys, "keys"), (values, "values")):
            strides = t.stride()
            if strides[3] != 1 or head_dim % part or t.data_ptr() % 16 or any(
                    n > 1 and (s < head_dim or s % part) for n, s in zip(t.shape[:3], strides)):
                raise ValueError(f"{name}: rows of whole 16 bytes, 16-byte aligned, one behind the other")
            ordered = sorted((s, n) for n, s in zip(t.shape[:3], strides) if n > 1)
            if any(big < s * n for (s, n), (big, _) in zip(ordered, ordered[1:])):
                raise ValueError(f"{name} must not overlap themselves")
        if _meet(keys, values):
            raise ValueError("keys and values must not share the same memory")
        for t, name in ((values, "values"), (table, "page_table"), (self.k_scale, "k_scale"), (self.v_scale, "v_scale")):
            if t is not None:
                _same_device(keys, t, name)
        for t, name in ((self.k_scale, "k_scale"), (self.v_scale, "v_scale")):
            if t is None:
                continue
            if keys.dtype == torch.bfloat16:
                raise ValueError(f"{name} goes with float8_e4m3fn caches")
            if t.dtype != torch.float32:
                raise TypeError(f"{name} must be float32")
            if t.shape != (kv_heads,) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous [{kv_heads}]")
        stride = lambda t: [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride())]  # noqa: E731
        (kp, kh, kt), (vp, vh, vt) = stride(keys), stride(values)
        object.__setattr__(self, "_struct", _lib.PagedCacheStruct(
            ptr(keys), ptr(values), _CACHE[keys.dtype], kv_heads, head_dim, page_size, pages, kp, kh, kt, vp, vh, vt,
            ptr(table), table.stride(0) if table.shape[0] > 1 else table.shape[1], table.shape[0], table.shape[1],
            ptr(self.k_scale), ptr(self.v_scale)))
        object.__setattr__(self, "_ref", ctypes.byref(self._struct))
        (k0, k1), (v0, v1) = _span(keys), _span(values)
        object.__setattr__(self, "_spans", (min(k0, v0), max(k1, v1), k0, k1, v0, v1))
        object.__setattr__(self, "_sizes", (_CACHE[keys.dtype], kv_heads, head_dim, page_size, table.shape[1]))

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int, max_pages: int,
              dtype: torch.dtype = torch.bfloat16, device="cuda", k_scale=None, v_scale=None) -> PagedCache:
        """A cache of ``pages`` pages, none of them mapped."""
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((slots, max_pages), -1, dtype=torch.int32, device=device), k_scale, v_scale)

    @property
    def device(self) -> torch.device:
        return self.keys.device


def _off_the_cache(cache: PagedCache, name: str, at: int, end: int) -> None:
    """Refuses bytes [at, end) that lie where the keys or the values do."""
    _, _, k0, k1, v0, v1 = cache._spans
    if at < k1 and end > k0 or at < v1 and end > v0:
        raise ValueError(f"{name} must not overlap the cache")


def append_paged(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                 row_slots: torch.Tensor, rope: Rope | None = None, q: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes ``k`` and ``v`` bf16 [T, kv_heads, head_dim] of new tokens to the
    cache, row r as token ``positions[r]`` of slot ``row_slots[r]`` (int32 or int64
    [T] each; a chunk's positions count what its slot holds already, as above), keys
    rotated by ``rope`` on the way.  With ``q`` bf16 [T, heads, head_dim], returns the rotated queries
    (into ``out``, which may be ``q``).  The three are usually views of one
    projection's rows; none of them lies in the cache.

    Rows of a slot outside [0, slots), of a negative position or one past the
    table, and of an unmapped page write nothing; their queries are rotated.  No
    two rows may name the same token: which of them it would hold is not said."""
    rows, kv_heads, dim, k_row, k_head, index = _heads(k, "k")
    v_rows, v_heads, v_dim, v_row, v_head, v_index = _heads(v, "v")
    _, cache_heads, head_dim, _, _ = cache._sizes
    if kv_heads != cache_heads or dim != head_dim or (v_rows, v_heads, v_dim) != (rows, kv_heads, dim):
        raise ValueError(f"k and v must be [T, {cache_heads}, {head_dim}], as the cache's heads")
    if v_index != index:
        _elsewhere(k, v, "v")
    if cache.keys.get_device() != index:
        _elsewhere(k, cache.keys, "cache")
    position_code = _indices(positions, "positions", rows, k, index)
    slot_code = _indices(row_slots, "row_slots", rows, k, index)
    # (what lies behind the cache needs no second look)
    low, high = cache._spans[:2]
    k_at, v_at = k.data_ptr(), v.data_ptr()
    if k_at < high and (end := k_at + 2 * ((rows - 1) * k_row + (kv_heads - 1) * k_head + dim)) > low:
        _off_the_cache(cache, "k", k_at, end)
    if v_at < high and (end := v_at + 2 * ((rows - 1) * v_row + (kv_heads - 1) * v_head + dim)) > low:
        _off_the_cache(cache, "v", v_at, end)
    rope_ref = None
    if rope is not None:
        rope_ref = rope._ref
        if rope.turns.get_device() != index:
            _elsewhere(k, rope.turns, "rope")
        if rope.rotary_dim > head_dim:
            raise ValueError(f"rotary width {rope.rotary_dim} above the head's {head_dim}")
    q_args = (None, 0, 0, 0, None, 0, 0)
    if q is not None:
        q_rows, heads, q_dim, q_row, q_head, q_index = _heads(q, "q")
        if q_rows != rows or q_dim != head_dim:
            raise ValueError(f"q must be [{rows}, heads, {head_dim}]")
        if q_index != index:
            _elsewhere(k, q, "q")
        q_at = q.data_ptr()
        if q_at < high and (end := q_at + 2 * ((rows - 1) * q_row + (heads - 1) * q_head + dim)) > low:
            _off_the_cache(cache, "q", q_at, end)
        if out is None:
            out = torch.empty(rows, heads, head_dim, dtype=q.dtype, device=q.device)
            out_row, out_head = heads * head_dim, head_dim
        else:
            _check_out(out, q, "out", True)
            if out.data_ptr() != q_at:
                if not (_apart(out, k) and _apart(out, v)):
                    raise ValueError("out must not overlap k or v")
                _off_the_cache(cache, "out", *_span(out))
            else:  # (in place: parts of one projection's rows, as a rule)
                extent, step = 2 * ((heads - 1) * q_head + dim), 2 * q_row
                for x, at, x_row, x_head in ((k, k_at, k_row, k_head), (v, v_at, v_row, v_head)):
                    beside = x_row == q_row > 0 and extent <= (at - q_at) % step <= step - 2 * ((kv_heads - 1) * x_head + dim)
                    if not beside and _meet(out, x):
                        raise ValueError("out must not overlap k or v")
            out_row, out_head, _ = out.stride()
        q_args = (q_at, q_row, q_head, heads, out.data_ptr(), out_row, out_head)
    elif out is not None:
        raise ValueError("out goes with q")
    _launch(index, "d3_paged_append", cache._ref, k_at, k_row, k_head, v_at, v_row, v_head, rows,
            positions.data_ptr(), position_code, row_slots.data_ptr(), slot_code, rope_ref, *q_args)
    return out


def paged_attention(q: torch.Tensor, cache: PagedCache, layout: PackedLayout, lengths: torch.Tensor,
                    scale: float | None = None, window: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens' queries ``q`` bf16 [T, heads, head_dim] over
    the cache -> bf16 [T, heads, head_dim].

    Rows ``[layout.boundaries[i], layout.boundaries[i + 1])`` are the newest tokens
    of sequence i, which slot ``layout.sequence_slots[i]`` holds ``lengths[i]`` tokens
    of, theirs included (int32 or int64 [n]; append first).  Row j of its n_i, at
    position ``p = lengths[i] - n_i + j``, attends the mapped tokens up to p, the
    last ``window`` of them where one is given, with weights
    ``softmax(scale * q . k)`` (``scale`` defaults to head_dim ** -0.5); query head h
    reads kv head ``h // (heads / kv_heads)``.  Rows that attend nothing are zeros; where
    all scores of a row are minus infinity, it is NaN.  A row's last bits may change with
    the rest of the batch, which how the call is cut follows.

    Rows of no sequence (before the first boundary, from the last on) are zeros, or
    left as they were in a given ``out`` (apart from ``q``).  ``layout.max_length`` is the
    longest n_i: 1 chooses the kernel for single tokens; any value computes all rows.
    head_dim is 64, 128 or 256."""
    rows, heads, dim, q_row, q_head, index = _heads(q, "q")
    boundaries, slots = layout.boundaries, layout.sequence_slots
    if boundaries.dtype != torch.int32:
        raise TypeError("boundaries must be int32")
    if boundaries.dim() != 1 or not boundaries.shape[0] or (boundaries.shape[0] > 1 and boundaries.stride(0) != 1):
        raise ValueError("boundaries must be contiguous [n + 1]")
    if boundaries.get_device() != index:
        _elsewhere(q, boundaries, "boundaries")
    count = boundaries.shape[0] - 1
    slot_code = _indices(slots, "sequence_slots", count, q, index)
    length_code = _indices(lengths, "lengths", count, q, index)
    sizes = cache._sizes
    if dim != sizes[2] or heads % sizes[1]:
        raise ValueError(f"q must be [T, heads, {sizes[2]}], heads a multiple of {sizes[1]}")
    if cache.keys.get_device() != index:
        _elsewhere(q, cache.keys, "cache")
    if window is not None and window < 1:
        raise ValueError(f"window {window} must be positive (or None)")
    if scale is None:
        scale = dim ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"scale {scale} must be finite")
    zero_rest = out is None
    if zero_rest:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
        out_row, out_head = heads * dim, dim
    else:
        _check_out(out, q, "out", False)
        _off_the_cache(cache, "out", *_span(out))
        out_row, out_head, _ = out.stride()
    longest = max(0, min(int(layout.max_length), _MOST))
    size = _workspace_bytes(sizes, rows, heads, count, longest)
    workspace, at = None, None
    if size > 0:
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        at = workspace.data_ptr()
    _launch(index, "d3_paged_attention", cache._ref, q.data_ptr(), q_row, q_head, rows, heads, boundaries.data_ptr(),
            slots.data_ptr(), slot_code, lengths.data_ptr(), length_code, count, longest, scale,
            0 if window is None else min(int(window), 1 << 62), out.data_ptr(), out_row, out_head, zero_rest, at, max(size, 0))
    return out
