// Attention of new tokens over a paged cache: arguments, and how the work of a
// call is cut, which every workgroup derives itself from the boundaries and
// lengths on the device (one captured call serves every batch).
//
// A sequence's new rows times the heads that share a kv head are packed rows:
// packed row m of kv head h is token m / group, query head h * group + m % group.
// They are cut into tiles of kTileRows; the keys a tile attends are cut into
// splits of whole 64-key blocks where one workgroup a tile would leave the card
// idle.  Unit = (tile, split); a workgroup takes one unit of one kv head.
#pragma once

#include "common.h"
#include "expert_tile.h"
#include "rows.h"

namespace d3 {

constexpr int kKeyBlock = 64;  // keys a split is cut at

struct PagedArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t out_row, out_head;
  const uint8_t *keys, *values;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  const int32_t* page_table;
  int64_t table_stride;
  uint32_t pages;
  int slots, page_shift;
  int capacity;  // tokens the table holds
  const float *k_scales, *v_scales;
  const int32_t* boundaries;
  const void *sequence_slots, *lengths;
  int slots_64, lengths_64;
  int sequences, rows, q_heads, kv_heads, group;
  int slices;       // 16-row parts of a token's group, each a tile of its own (decode)
  int tile_rows;    // packed rows of a tile, or 0: one token's slice (decode)
  int tile_tokens;  // most tokens a tile spans
  float scale;      // with log2(e) in it: weights are powers of two
  int window;       // 0: none
  int target;       // units a kv head that the splits aim at
  int least;        // fewest key blocks worth a split
  int max_units;    // of a kv head, bounds the grid
  int zero_rest;
  float* sums;      // partial rows [split unit][kv head][tile rows][D]
  float2* stats;    // their (maximum, sum) [split unit][kv head][tile rows]
};

// One unit's place.
struct PagedUnit {
  bool live;
  int sequence, tile, split, splits, partial;  // partial: first partial of the tile's splits, where splits > 1
  int first_row, tokens, length;               // rows of the sequence, tokens it holds
};

struct PagedSequence {
  int first_row, tokens, length, tiles, splits, blocks;
};

__device__ __forceinline__ int64_t paged_index(const void* p, int is_64, int64_t i) {
  return is_64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ PagedSequence paged_sequence(const PagedArgs& a, int i) {
  PagedSequence s = {};
  if (i >= a.sequences) return s;
  const int b0 = min(max(a.boundaries[i], 0), a.rows), b1 = min(max(a.boundaries[i + 1], 0), a.rows);
  const int64_t length = paged_index(a.lengths, a.lengths_64, i);
  s.first_row = b0;
  s.tokens = max(b1 - b0, 0);
  s.length = static_cast<int>(length < 0 ? 0 : (length < 0x7fffffff ? length : 0x7fffffff));
  s.tiles = a.tile_rows ? (s.tokens * a.group + a.tile_rows - 1) / a.tile_rows : s.tokens * a.slices;
  // Key blocks of the longest tile: all the sequence's, or what a window over its tokens touches.
  int keys = min(s.length, a.capacity);
  if (a.window > 0) keys = static_cast<int>(min(static_cast<int64_t>(keys), static_cast<int64_t>(a.window) + a.tile_tokens + kKeyBlock));
  s.blocks = (keys + kKeyBlock - 1) / kKeyBlock;
  return s;
}

__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(wave_reduce<SumF32>(__float_as_uint(v)));
}

// Inclusive prefix sum over the wave's lanes.
__device__ __forceinline__ int wave_prefix(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(v, d, kWave);
    if (lane_id() >= d) v += up;
  }
  return v;
}

// Key blocks of a split: the batch's blocks over the units aimed at.  A little
// more than their quotient, so that the units stay within tiles + target
// whatever fp32 rounds off.
__device__ __forceinline__ int paged_chunk(const PagedArgs& a) {
  float work = 0.0f;
  for (int i = lane_id(); i - lane_id() < a.sequences; i += kWave) {
    const PagedSequence s = paged_sequence(a, i);
    work += static_cast<float>(s.tiles) * static_cast<float>(s.blocks);
  }
  work = wave_sum(work);
  const float chunk = ceilf(work * 1.001f / static_cast<float>(a.target));
  return max(a.least, chunk < 1e9f ? static_cast<int>(chunk) : 1000000000);
}

// The unit with index `at`, found by every wave for itself (no barrier); with
// kTiles, the tile with index `at` among those that are split.
template <bool kTiles>
__device__ __forceinline__ PagedUnit paged_unit(const PagedArgs& a, int at) {
  const int chunk = paged_chunk(a);
  int units_before = 0, partials_before = 0;
  for (int base = 0; base < a.sequences; base += kWave) {
    PagedSequence s = paged_sequence(a, base + lane_id());
    s.splits = max(1, (s.blocks + chunk - 1) / chunk);
    const int units = kTiles ? (s.splits > 1 ? s.tiles : 0) : s.tiles * s.splits;
    const int partials = s.splits > 1 ? s.tiles * s.splits : 0;
    const int units_to = units_before + wave_prefix(units);
    const int partials_to = partials_before + wave_prefix(partials);
    const uint64_t here = __ballot(at < units_to);
    if (here != 0) {
      const int lane = __builtin_ctzll(here);
      PagedUnit u;
      u.live = true;
      u.sequence = base + lane;
      u.splits = __builtin_amdgcn_readlane(s.splits, lane);
      u.first_row = __builtin_amdgcn_readlane(s.first_row, lane);
      u.tokens = __builtin_amdgcn_readlane(s.tokens, lane);
      u.length = __builtin_amdgcn_readlane(s.length, lane);
      const int tiles = __builtin_amdgcn_readlane(s.tiles, lane);
      const int rest = at - (__builtin_amdgcn_readlane(units_to, lane) - __builtin_amdgcn_readlane(units, lane));
      // The last tile attends the most keys: it comes first.
      u.tile = tiles - 1 - (kTiles ? rest : rest / u.splits);
      u.split = kTiles ? 0 : rest % u.splits;
      u.partial = __builtin_amdgcn_readlane(partials_to, lane) - __builtin_amdgcn_readlane(partials, lane) +
                  u.tile * u.splits;
      return u;
    }
    units_before = __builtin_amdgcn_readlane(units_to, kWave - 1);
    partials_before = __builtin_amdgcn_readlane(partials_to, kWave - 1);
  }
  PagedUnit none = {};
  return none;
}

// Keys [low, high) that a split of a tile attends: of tokens [first, last] of
// the sequence, in whole blocks from the tile's first key's block.
struct PagedKeys {
  int low, high;
};
__device__ __forceinline__ PagedKeys paged_keys(const PagedArgs& a, const PagedUnit& u, int first, int last) {
  const int before = u.length - u.tokens;  // may be negative: rows with no place
  const int end = min(max(before + last + 1, 0), a.capacity);
  const int64_t seen = a.window > 0 ? static_cast<int64_t>(before) + first - a.window + 1 : 0;
  const int start = static_cast<int>(seen > 0 ? (seen < end ? seen : end) : 0);
  const int aligned = start & ~(kKeyBlock - 1);
  const int blocks = (end - aligned + kKeyBlock - 1) / kKeyBlock;
  const int each = (blocks + u.splits - 1) / u.splits;
  PagedKeys k;
  const int64_t from = aligned + static_cast<int64_t>(u.split) * each * kKeyBlock;
  const int64_t to = from + static_cast<int64_t>(each) * kKeyBlock;
  k.low = static_cast<int>(from > start ? (from < end ? from : end) : start);
  k.high = static_cast<int>(to < end ? to : end);
  if (k.high < k.low) k.high = k.low;
  return k;
}

// Rows before the first sequence and behind the last are zeroed, a row a workgroup.
__device__ __forceinline__ void paged_zero_rest(const PagedArgs& a, int workgroup, int workgroups, int head_dim) {
  const int b0 = a.sequences > 0 ? min(max(a.boundaries[0], 0), a.rows) : a.rows;
  const int b1 = a.sequences > 0 ? max(min(max(a.boundaries[a.sequences], 0), a.rows), b0) : a.rows;
  const int rest = b0 + a.rows - b1;
  for (int r = workgroup; r < rest; r += workgroups) {
    uint16_t* row = a.out + (r < b0 ? r : b1 + r - b0) * a.out_row;
    for (int i = static_cast<int>(threadIdx.x); i < a.q_heads * head_dim; i += static_cast<int>(blockDim.x))
      row[(i / head_dim) * a.out_head + i % head_dim] = 0;
  }
}

// A row of zeros: where tokens that no row attends are read from instead.
static __device__ __attribute__((aligned(16))) uint8_t paged_nothing[512];

typedef short int16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

// Transposing LDS read of 16-bit values: each 16-lane group reads four rows of
// 16 columns, lane i row i / 4, columns 4 (i % 4) .. + 4; lane i gets column i of
// the four rows.
__device__ __forceinline__ uint32x2 read_transposed(const uint8_t* at) {
  return __builtin_bit_cast(uint32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                          (__attribute__((address_space(3))) int16x4*)(at)));
}

__device__ __forceinline__ bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const int32x4 w = {static_cast<int>(a), static_cast<int>(b), static_cast<int>(c), static_cast<int>(d)};
  return __builtin_bit_cast(bf16x8, w);
}

// 8 e4m3 codes to bf16, exactly.
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Maximum and sum with the lane 32 away, and with those 16 and 32 away, in every lane.
__device__ __forceinline__ float max_across_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_across_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_across_32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_across_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_across_32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// 2^x by the hardware's v_exp_f32; -inf gives 0.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four consecutive columns of a row, rounded.
typedef uint32_t RowVector2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ void store_row4(uint16_t* out, floatx4 v) {
  *reinterpret_cast<RowVector2*>(out) = RowVector2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

void launch_paged_decode(const PagedArgs& a, int head_dim, bool e4m3, hipStream_t stream);
void launch_paged_tiles(const PagedArgs& a, int head_dim, bool e4m3, hipStream_t stream);

}  // namespace d3
