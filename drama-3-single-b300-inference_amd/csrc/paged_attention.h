// Attention of new tokens over a paged cache: arguments, and how the work of a
// call is cut, which every workgroup derives itself from the boundaries and
// lengths on the device (one captured call serves every batch).
//
// A sequence's new rows times the heads that share a kv head are packed rows:
// packed row m of kv head h is token m / group, query head h * group + m % group.
// They are cut into tiles of 128 or 256, a sequence's single token into one tile per
// 16 heads of its group.
//
// Single tokens: the key blocks of all their tiles, one behind the other, are dealt
// to as many workgroups as are resident at once, the same number to each; where a
// workgroup's share ends inside a tile, the tile's parts are joined afterwards.
// Tiles of many rows: a workgroup each, or several for those of more key blocks
// than an even share.
#pragma once

#include <type_traits>

#include "common.h"
#include "expert_tile.h"
#include "rows.h"

namespace d3 {

constexpr int kKeyBlock = 64;  // keys that tiles are cut at
constexpr int kLeastSplit = 4;   // fewest key blocks worth a split of a tile
constexpr int kGroupRows = 128;  // packed rows that four waves of a tile take
constexpr float kLog2E = 1.4426950408889634f;
constexpr int kZeroGroups = 64;  // workgroups behind the units' that zero rows of no sequence

struct PagedArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t out_row, out_head;
  const uint8_t *keys, *values;
  uint32_t k_page, k_token, v_page, v_token;  // bytes: products with a page's number are one instruction
  int64_t k_head, v_head;
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
  int slices;         // 16-row parts of a token's group, each a tile where tokens are taken singly
  int all_single;     // every token is taken singly (else those of sequences of one)
  int tile_rows;      // packed rows of the other tiles
  int tile_tokens;    // most tokens a tile spans
  float scale;        // with log2(e) in it: weights are powers of two
  int window;         // 0: none
  int share_shift;    // log2 of the keys in a block of single tokens' shares
  int shares, least;  // workgroups a kv head that single tokens' blocks are dealt to, fewest blocks of one
  int target;         // units a kv head that the splits of tiles aim at
  uint32_t target_inverse;  // 2^32 / target, rounded up: a high product with it is the quotient or one more
  int work_shift;     // log2 of the blocks in one of their sums, which stay below 2^31
  int splitting;      // whether they may be split
  int tile_units;     // most units of a kv head
  // Partial rows [part][kv head][rows of a tile][D] and their (maximum, sum), of single
  // tokens' tiles (16 rows) and of the others (tile_rows).
  float *single_sums, *tile_sums;
  float2 *single_stats, *tile_stats;
  // A workgroup's share has two of the former at most (PagedShares).
  int tile_parts;  // how many there are: boundaries that are not ascending must not lead past them
};

// Where a workgroup's work lies.
struct PagedUnit {
  bool live;
  int tile, splits;
  int split;                      // of a tile: which of its splits
  int from, blocks;               // of a single token's tile: blocks [from, from + blocks)
  int part;                       // partial of this unit (of a tile to join: the first)
  int first_row, tokens, length;  // rows of the sequence, tokens it holds
  int slot;                       // [0, slots), or -1
};

struct PagedSequence {
  int first_row, tokens, length, slot, tiles, blocks;
  bool single;
};

__device__ __forceinline__ int64_t paged_index(const void* p, int is_64, int64_t i) {
  return is_64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ PagedSequence paged_sequence(const PagedArgs& a, int i) {
  // (loads of every lane at once, none behind another)
  const int at = min(i, a.sequences - 1);
  const int from = a.boundaries[at], to = a.boundaries[at + 1];
  const int64_t length = paged_index(a.lengths, a.lengths_64, at);
  const int64_t slot = paged_index(a.sequence_slots, a.slots_64, at);
  const int b0 = min(max(from, 0), a.rows), b1 = min(max(to, 0), a.rows);
  PagedSequence s;
  s.first_row = b0;
  s.tokens = i < a.sequences ? max(b1 - b0, 0) : 0;
  s.length = static_cast<int>(length < 0 ? 0 : (length < 0x7fffffff ? length : 0x7fffffff));
  s.slot = slot >= 0 && slot < a.slots ? static_cast<int>(slot) : -1;
  s.single = a.all_single || s.tokens == 1;
  s.tiles = s.single ? s.tokens * a.slices : static_cast<int>(static_cast<uint32_t>(s.tokens * a.group + a.tile_rows - 1) / static_cast<uint32_t>(a.tile_rows));
  // Key blocks of the longest tile: all the sequence's, or what a window over its tokens touches.
  int keys = min(s.length, a.capacity);
  const int shift = s.single ? a.share_shift : 6;
  if (a.window > 0)
    keys = static_cast<int>(min(static_cast<int64_t>(keys), static_cast<int64_t>(a.window) + a.tile_tokens + (1 << shift)));
  s.blocks = max((keys + (1 << shift) - 1) >> shift, 1);
  return s;
}

__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(wave_reduce<SumF32>(__float_as_uint(v)));
}

// Inclusive prefix sum over the wave's lanes, on DPP moves: within rows of 16, then rows' ends.
__device__ __forceinline__ int wave_prefix(int value) {
  uint32_t v = static_cast<uint32_t>(value);
  v += dpp_move<0x111>(v, 0);  // row_shr 1, 2, 4, 8
  v += dpp_move<0x112>(v, 0);
  v += dpp_move<0x114>(v, 0);
  v += dpp_move<0x118>(v, 0);
  v += dpp_move<kDppRowBcast15, 0xa>(v, 0);
  v += dpp_move<kDppRowBcast31, 0xc>(v, 0);
  return static_cast<int>(v);
}

__device__ __forceinline__ int wave_total(int v) {
  return static_cast<int>(wave_reduce<SumU32>(static_cast<uint32_t>(v)));
}
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, kWave - 1); }

// A walk over the sequences, 64 at a time (a lane each), found by every wave for
// itself, without a barrier.
struct PagedWalk {
  PagedSequence mine;  // this lane's of the sequences [base, base + 64)
  int base;
  __device__ void start(const PagedArgs& a) { base = 0, mine = paged_sequence(a, lane_id()); }
  __device__ bool next(const PagedArgs& a) {
    base += kWave;
    if (base >= a.sequences) return false;
    mine = paged_sequence(a, base + lane_id());
    return true;
  }
  __device__ void take(int lane, PagedUnit& u) const {
    u.live = true;
    u.first_row = __builtin_amdgcn_readlane(mine.first_row, lane);
    u.tokens = __builtin_amdgcn_readlane(mine.tokens, lane);
    u.length = __builtin_amdgcn_readlane(mine.length, lane);
    u.slot = __builtin_amdgcn_readlane(mine.slot, lane);
  }
};

// Shares of single tokens' blocks: workgroup w of a kv head takes the blocks [w *
// each, (w + 1) * each) of all tiles one behind the other.  Part 2 w is what it
// computes of a tile that the share begins within, 2 w + 1 of one that begins in the share
// and ends behind it: a tile's first part is 2 w + 1 of its first workgroup, the others
// follow as 2 (w + 1), 2 (w + 2) ...
struct PagedShares {
  PagedWalk walk;
  int to, tiles_to;              // inclusive prefix sums over the walk's lanes
  int before, tiles_before;      // blocks and tiles before the walk's sequences
  int total, each;
  __device__ int blocks_here() const { return walk.mine.single ? walk.mine.tiles * walk.mine.blocks : 0; }
  __device__ int tiles_here() const { return walk.mine.single ? walk.mine.tiles : 0; }
  __device__ void sums() { to = before + wave_prefix(blocks_here()), tiles_to = tiles_before + wave_prefix(tiles_here()); }
  __device__ void start(const PagedArgs& a) {
    walk.start(a);
    before = tiles_before = 0;
    sums();
    total = last_lane(to);
    if (a.sequences > kWave) {
      while (walk.next(a)) total += wave_total(blocks_here());
      walk.start(a);
    }
    each = max(a.least, static_cast<int>((static_cast<uint32_t>(total) + a.shares - 1) / static_cast<uint32_t>(a.shares)));
  }
  // The tile that holds block `at` < total, of those from the walk's place on; u.from
  // is the block's place in it, u.blocks what it has from there.
  // kTiles: the tile with number `at`; u.from is its first block.
  template <bool kTiles = false>
  __device__ PagedUnit find(const PagedArgs& a, int at) {
    PagedUnit u = {};
    for (;;) {
      const uint64_t here = __ballot(at < (kTiles ? tiles_to : to));
      if (here != 0) {
        const int lane = __builtin_ctzll(here);
        walk.take(lane, u);
        const int blocks = __builtin_amdgcn_readlane(walk.mine.blocks, lane), tiles = __builtin_amdgcn_readlane(walk.mine.tiles, lane);
        const int first = __builtin_amdgcn_readlane(to, lane) - blocks * tiles;
        if constexpr (kTiles) {
          u.tile = at - (__builtin_amdgcn_readlane(tiles_to, lane) - tiles);
          u.from = first + u.tile * blocks, u.blocks = blocks;
          u.live = static_cast<uint32_t>(u.tile) < static_cast<uint32_t>(tiles);
          return u;
        }
        const uint32_t rest = static_cast<uint32_t>(at - first);
        u.tile = static_cast<int>(rest / static_cast<uint32_t>(blocks));
        u.from = static_cast<int>(rest) - u.tile * blocks;
        u.blocks = blocks - u.from;
        u.live = static_cast<uint32_t>(u.tile) < static_cast<uint32_t>(tiles);  // (sums of boundaries that do not ascend may wrap)
        return u;
      }
      before = last_lane(to), tiles_before = last_lane(tiles_to);
      if (!walk.next(a)) return u;
      sums();
    }
  }
};

// The unit with index `at` of the tiles of many rows; with kTiles, the tile with
// index `at` among those that are split.
template <bool kTiles>
__device__ __forceinline__ PagedUnit paged_tile_unit(const PagedArgs& a, int at) {
  PagedWalk walk;
  walk.start(a);
  auto tiles_here = [&] { return walk.mine.single ? 0 : walk.mine.tiles; };
  // Key blocks of a split: the batch's blocks over the units aimed at, so that the units
  // stay within tiles + target.  In integers: the tiles and their join each find it for
  // themselves, and have to find the same.
  auto work_here = [&] {
    return static_cast<uint32_t>(tiles_here()) * (static_cast<uint32_t>(walk.mine.blocks + (1 << a.work_shift) - 1) >> a.work_shift);
  };
  uint32_t work = wave_reduce<SumU32>(work_here());
  if (a.sequences > kWave) {
    while (walk.next(a)) work += wave_reduce<SumU32>(work_here());
    walk.start(a);
  }
  const uint32_t rounded_up = __umulhi(work + static_cast<uint32_t>(a.target) - (a.target > 1 ? 1 : 0), a.target_inverse);
  const int even = static_cast<int>(min(rounded_up, (1u << 30) >> a.work_shift)) << a.work_shift;
  // Fewest blocks worth a split: kLeastSplit where the units are few, else twice that.
  const int least = !a.splitting ? 1 << 30 : (even > 1 ? 2 * kLeastSplit : kLeastSplit);
  const int chunk = max(least, even);
  int units_before = 0, parts_before = 0;
  PagedUnit u = {};
  do {
    const int tiles = tiles_here();
    const int splits = static_cast<int>((static_cast<uint32_t>(walk.mine.blocks) + chunk - 1) / static_cast<uint32_t>(chunk));
    const int units = kTiles ? (splits > 1 ? tiles : 0) : tiles * splits;
    const int parts = splits > 1 ? tiles * splits : 0;
    const int units_to = units_before + wave_prefix(units);
    const int parts_to = parts_before + wave_prefix(parts);
    const uint64_t here = __ballot(at < units_to);
    if (here != 0) {
      const int lane = __builtin_ctzll(here);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, lane); };
      walk.take(lane, u);
      u.splits = of(splits);
      const uint32_t rest = static_cast<uint32_t>(at - (of(units_to) - of(units))), count = static_cast<uint32_t>(u.splits);
      // The last tile attends the most keys: it comes first.
      u.tile = of(tiles) - 1 - static_cast<int>(kTiles ? rest : rest / count);
      u.split = kTiles ? 0 : static_cast<int>(rest % count);
      u.part = of(parts_to) - of(parts) + u.tile * u.splits + u.split;
      u.live = static_cast<uint32_t>(u.tile) < static_cast<uint32_t>(of(tiles)) &&
               (u.splits <= 1 || (u.part >= 0 && u.part <= a.tile_parts - (kTiles ? u.splits : 1)));
      return u;
    }
    units_before = last_lane(units_to), parts_before = last_lane(parts_to);
  } while (walk.next(a));
  return u;
}

// Keys [low, high) of blocks [from, from + blocks) of a tile: of what tokens
// [first, last] of the sequence attend, counted from the first key's block.
struct PagedKeys {
  int low, high;
};
struct PagedReach {
  int start, end, aligned;  // keys [start, end), the first one's block's first key
};
__device__ __forceinline__ PagedReach paged_reach(const PagedArgs& a, const PagedUnit& u, int first, int last, int shift) {
  const int before = u.length - u.tokens;  // may be negative: rows with no place
  PagedReach r;
  r.end = u.slot < 0 ? 0 : min(max(before + last + 1, 0), a.capacity);
  const int64_t seen = a.window > 0 ? static_cast<int64_t>(before) + first - a.window + 1 : 0;
  r.start = static_cast<int>(seen > 0 ? (seen < r.end ? seen : r.end) : 0);
  r.aligned = r.start >> shift << shift;
  return r;
}
__device__ __forceinline__ PagedKeys paged_keys(const PagedReach& r, int from, int blocks, int shift) {
  const int64_t low = r.aligned + (static_cast<int64_t>(from) << shift), high = low + (static_cast<int64_t>(blocks) << shift);
  PagedKeys k;
  k.low = static_cast<int>(low > r.start ? (low < r.end ? low : r.end) : r.start);
  k.high = static_cast<int>(high < r.end ? high : r.end);
  if (k.high < k.low) k.high = k.low;
  return k;
}

// Rows before the first sequence and behind the last are zeroed, by workgroups of their own.
__device__ __forceinline__ void paged_zero_rest(const PagedArgs& a, int workgroup, int head_dim) {
  const int b0 = a.sequences > 0 ? min(max(a.boundaries[0], 0), a.rows) : a.rows;
  const int b1 = a.sequences > 0 ? max(min(max(a.boundaries[a.sequences], 0), a.rows), b0) : a.rows;
  const int rest = b0 + a.rows - b1;
  for (int r = workgroup; r < rest; r += kZeroGroups) {
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

// An address that another lane holds: of a lane known to the wave, and of any.
__device__ __forceinline__ const uint8_t* lane_address(const uint8_t* mine, int lane) {
  const uint64_t p = reinterpret_cast<uint64_t>(mine);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(p), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(p >> 32), lane);
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ const uint8_t* shuffled_address(const uint8_t* mine, int lane) {
  const uint64_t p = reinterpret_cast<uint64_t>(mine);
  const uint32_t lo = __shfl(static_cast<int>(p), lane, kWave), hi = __shfl(static_cast<int>(p >> 32), lane, kWave);
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(hi) << 32 | lo);
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

// What scores of a head are multiplied by, positive: a weight is 2^(score * size -
// maximum), one instruction before the exponential, and a masked score of -inf stays
// -inf.  A negative factor turns the query's signs instead, 0 is the least positive.
struct ScoreScale {
  float size;
  uint32_t sign;  // of both halves of a word of queries
};
__device__ __forceinline__ ScoreScale score_scale(float c) {
  return {c == 0.0f ? 1.17549435e-38f : fabsf(c), c < 0.0f ? 0x80008000u : 0u};
}
__device__ __forceinline__ bf16x8 load_query(const uint16_t* q, uint32_t sign) {
  const RowVector4 w = *reinterpret_cast<const RowVector4*>(q);
  return operand(w[0] ^ sign, w[1] ^ sign, w[2] ^ sign, w[3] ^ sign);
}

// 2^x by the hardware's v_exp_f32; -inf gives 0.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's weights are 2^(score * size - base), the product exact within one instruction, base
// the highest score times size, rounded.  The highest score's exponent is that rounding: at
// bases of 2^32 up to 2^8.  From kCoarse on (a step of 1) scores are therefore multiplied
// and rounded first, as the base was (and size is 1): the highest weighs 1, the others are
// off by half a step of theirs, as the fp32 scores are themselves.
//
// All that an ordinary block needs is whether its highest score is within the row's limit: NaN,
// which nothing is within, until the row attends a key; minus infinity where scores are
// coarse.  A row whose scores are all minus infinity has the lowest number as its base and
// weights of 0 / 0 (NaN); one that attends nothing keeps its limit (zeros).
constexpr float kCoarse = 8388608.0f, kLowest = -3.402823466e38f;

// Four consecutive columns of a row, rounded.
typedef uint32_t RowVector2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ void store_row4(uint16_t* out, floatx4 v) {
  *reinterpret_cast<RowVector2*>(out) = RowVector2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// A workgroup that no unit takes: the rows of no sequence, zeroed.
inline unsigned paged_workgroups(const PagedArgs& a, bool zero_rest) {
  return static_cast<unsigned>((a.tile_units + a.shares) * a.kv_heads + (zero_rest ? kZeroGroups : 0));
}

void launch_paged_decode(const PagedArgs& a, int head_dim, bool e4m3, bool zero_rest, hipStream_t stream);

}  // namespace d3
