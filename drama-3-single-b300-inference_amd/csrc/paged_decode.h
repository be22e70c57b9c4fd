// Attention of single new tokens over a paged cache, one pass over the keys.
//
// The query heads of one token that share a kv head (up to 16) are the columns
// of mfma_f32_16x16x32_bf16; keys are its rows: S^T = K Q^T leaves a lane 4 keys
// of one head per tile, so maximum, sum and rescale of the running softmax stay
// in the lane's own column, and O^T = V^T P^T takes P^T as it lies in registers
// once keys are numbered 16 (j / 4) + 4 g + j % 4 (lane group g, element j) in
// both operands.  Keys come from memory straight into operand registers; values
// go through LDS, whose transposing reads give four keys of one column.
//
// Bound by HBM: every key and value is read once.  The waves of a workgroup
// take steps of 32 keys in turn, each with its own running softmax and no
// barrier until the end, where their rows are added in LDS; the next step's
// keys and values are in flight while one is multiplied.  16 tokens over 32768 e4m3
// keys 134 us (6.2 TB/s); 52 over 2048 keys of 256 columns 39.0 (34 and the join of the
// parts); a token's 333 keys 8.1: three dependent loads of the plan, then steps of 128 keys in turn.
#pragma once

#include "paged_attention.h"

namespace d3 {

// Keys of a wave's step: what its registers hold twice (rows of 256 columns: half, for two waves a SIMD).
constexpr int decode_keys(int dim) { return dim == 256 ? 16 : 32; }

// Keys and values are read once: past the caches' use for them (16 x 32768 e4m3 keys
// 151 us, 171 as ordinary loads).
__device__ __forceinline__ int32x4 load_once(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const int32x4*>(p));
}

template <int D, int kWaves>
struct DecodeShared {
  // a wave's values, later its fp32 rows of 16 columns
  __attribute__((aligned(16))) uint8_t values[kWaves][16 * D * 4];
  float2 stats[kWaves][16];
};

template <int D, bool kE4m3, int kWaves>
__device__ __forceinline__ void decode_unit(const PagedArgs& a, const PagedUnit& u, int head, DecodeShared<D, kWaves>& shared) {
  constexpr int kKeys = decode_keys(D), kKeyTiles = kKeys / 16;
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowParts = D * kBytes / 16;              // 16-byte parts of a cached row
  constexpr int kKeyLoads = kKeyTiles * (kRowParts / 4);  // a lane's: key lane % 16 of the tiles, every fourth part
  constexpr int kKeysALoad = kWave / kRowParts;           // value rows a load covers
  constexpr int kValueLoads = kKeys / kKeysALoad;
  constexpr int kSteps = D / 32, kTiles = D / 16;
  constexpr int kSwizzle = D >= 128 ? 7 : 3;
  constexpr int kShift = D >= 128 ? 0 : 1;
  int lane = lane_id();
  asm volatile("" : "+v"(lane));  // (nothing of a unit's is held in registers over a share's other units)
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int column = lane & 15, g = lane >> 4;
  const int token = u.tile / a.slices, slice = u.tile % a.slices;
  const int heads = min(16, a.group - 16 * slice);  // live columns
  const int row = u.first_row + token;
  const int q_head0 = head * a.group + 16 * slice;
  const ScoreScale scale = score_scale(a.scale * (kE4m3 && a.k_scales != nullptr ? a.k_scales[head] : 1.0f));

  // Q^T operand: column = head, elements by the keys' order of the contraction.
  // bf16 keys: step s, element j of group g is column 32 s + 8 g + j; e4m3 ones
  // come 16 at a time: 64 (s / 2) + 16 g + 8 (s % 2) + j.
  bf16x8 qf[kSteps];
  {
    const uint16_t* q = a.q + row * a.q_row + (q_head0 + min(column, heads - 1)) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = kE4m3 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      qf[s] = load_query(q + d, scale.sign);
    }
  }
  const PagedKeys range = paged_keys(paged_reach(a, u, token, token, a.share_shift), u.from, u.blocks, a.share_shift);
  const int32_t* pages = a.page_table + (u.slot < 0 ? 0 : u.slot) * a.table_stride;
  const uint8_t* keys = a.keys + head * a.k_head;
  const uint8_t* values = a.values + head * a.v_head;
  const int in_page = (1 << a.page_shift) - 1;

  floatx4 o[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) o[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  float base = 0.0f, limit = __builtin_nanf(""), size = scale.size, sum = 0.0f;

  // Steps from the aligned one that holds the first key; wave w takes every kWaves-th.
  const int first = range.low & ~(kKeys - 1);
  // The page of a step's key `lane`: the table's entry, loaded a step before it is
  // looked at (a use waits for every load before it); then -1 where nothing is attended.
  auto attends = [&](int key) { return key + (lane & (kKeys - 1)) >= range.low && key + (lane & (kKeys - 1)) < range.high; };
  auto entry_of = [&](int key) { return pages[attends(key) ? (key + (lane & (kKeys - 1))) >> a.page_shift : 0]; };
  auto page_of = [&](int key, int entry) { return attends(key) && static_cast<uint32_t>(entry) < a.pages ? entry : -1; };
  int32x4 kr[kKeyLoads], vr[kValueLoads];
  // (a lane works out where its own key's rows begin, the loads take it from there)
  auto load_keys = [&](int key, int page) {
    const uint64_t token = (key + lane % kKeys) & in_page, p = static_cast<uint32_t>(page);
    const uint8_t* row = page < 0 ? paged_nothing : keys + (p * a.k_page + token * a.k_token);
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t) {
      const uint8_t* at = shuffled_address(row, 16 * t + column) + 16 * g;
#pragma unroll
      for (int i = 0; i < kRowParts / 4; ++i)
        kr[t * (kRowParts / 4) + i] = load_once(at + 64 * i);
    }
  };
  auto load_rows = [&](int key, int page) {
    const uint64_t token = (key + lane % kKeys) & in_page, p = static_cast<uint32_t>(page);
    const uint8_t* row = page < 0 ? paged_nothing : values + (p * a.v_page + token * a.v_token);
#pragma unroll
    for (int i = 0; i < kValueLoads; ++i)
      vr[i] = load_once(shuffled_address(row, kKeysALoad * i + lane / kRowParts) + 16 * (lane % kRowParts));
  };

  int key = first + wave * kKeys;
  int page = page_of(key, entry_of(key));
  int entry = entry_of(key + kWaves * kKeys);
  if (key < range.high) {
    load_keys(key, page);
    load_rows(key, page);
  }
  uint8_t* mine = shared.values[wave];
  for (; key < range.high; key += kWaves * kKeys) {
    const uint32_t attended = static_cast<uint32_t>(__ballot(page >= 0)) & (kKeys == 32 ? 0xffffffffu : 0xffffu);
    // S^T of the step's 16-key tiles
    floatx4 s[kKeyTiles];
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t) {
      s[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kRowParts / 4; ++i) {
        const int32x4 w = kr[t * (kRowParts / 4) + i];
        if constexpr (kE4m3) {
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[0], w[1]), qf[2 * i], s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[2], w[3]), qf[2 * i + 1], s[t], 0, 0, 0);
        } else {
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), qf[i], s[t], 0, 0, 0);
        }
      }
    }
    const int next = key + kWaves * kKeys;
    const int next_page = page_of(next, entry);
    entry = entry_of(next + kWaves * kKeys);
    if (next < range.high) load_keys(next, next_page);
    // The running softmax, in powers of two
    if (attended != (kKeys == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
      for (int t = 0; t < kKeyTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][i] = (attended >> (16 * t + 4 * g + i)) & 1u ? s[t][i] : -__builtin_huge_valf();
    }
    float most = s[0][0];
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, s[t][i]);
    most = max_across_16(most) * scale.size;
    if (__any(!(most <= limit))) {
      const bool fresh = limit != limit, attends = attended != 0;
      const bool raise = fresh ? attends : most > base;
      const float higher = raise ? fmaxf(most, kLowest) : base;
      const float shrink = raise && !fresh ? exp2_fast(base - higher) : 1.0f;
      base = higher;
      sum *= shrink;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] *= shrink;
      const bool coarse = __any(fabsf(base) >= kCoarse);
      if (!fresh || attends) limit = coarse ? -__builtin_huge_valf() : base;
      size = coarse ? 1.0f : scale.size;
      if (coarse) {
#pragma unroll
        for (int t = 0; t < kKeyTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][i] *= scale.size;
      }
    }
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = exp2_fast(fmaf(s[t][i], size, -base));
        sum += s[t][i];
      }
    uint32_t p[2 * kKeyTiles];
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t)
      p[2 * t] = pack_bf16x2(s[t][0], s[t][1]), p[2 * t + 1] = pack_bf16x2(s[t][2], s[t][3]);
    // Values to the wave's LDS: 16-byte part c of row r at c ^ 2 (r % 8) (D = 64: by
    // pairs of rows), so that the 32-byte pieces of eight rows fall on all banks.
#pragma unroll
    for (int i = 0; i < kValueLoads; ++i) {
      const int r = kKeysALoad * i + lane / kRowParts;
      const int turn = 2 * ((r >> kShift) & kSwizzle);
      if constexpr (kE4m3) {
        const int c = 2 * (lane % kRowParts);
        *reinterpret_cast<bf16x8*>(mine + r * (2 * D) + ((c ^ turn) << 4)) = widen8(vr[i][0], vr[i][1]);
        *reinterpret_cast<bf16x8*>(mine + r * (2 * D) + (((c + 1) ^ turn) << 4)) = widen8(vr[i][2], vr[i][3]);
      } else {
        *reinterpret_cast<int32x4*>(mine + r * (2 * D) + (((lane % kRowParts) ^ turn) << 4)) = vr[i];
      }
    }
    if (next < range.high) load_rows(next, next_page);
    page = next_page;
    // O^T += V^T P^T
    const int r = 4 * g + (column >> 2);
    const int turn = 2 * ((r >> kShift) & kSwizzle);  // row r + 16 has the same
    const uint8_t* at = mine + r * (2 * D) + 8 * (column & 1);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int part = ((2 * t + ((column >> 1) & 1)) ^ turn) << 4;
      const uint32x2 lo = read_transposed(at + part);
      if constexpr (kKeys == 32) {
        const uint32x2 hi = read_transposed(at + part + 16 * 2 * D);
        o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(lo[0], lo[1], hi[0], hi[1]), operand(p[0], p[1], p[2], p[3]),
                                                       o[t], 0, 0, 0);
      } else {
        o[t] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(int16x4, lo),
                                                         __builtin_bit_cast(int16x4, uint32x2{p[0], p[1]}), o[t], 0, 0, 0);
      }
    }
  }

  // The waves' rows to LDS (fp32 [column][D], a wave's values' space), then one
  // pass adds them at the weights of their maxima.
  sum = sum_across_16(sum);
  if (g == 0) shared.stats[wave][column] = make_float2(limit != limit ? -__builtin_huge_valf() : base, sum);
  float* sums = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
    *reinterpret_cast<floatx4*>(sums + column * D + ((16 * t + 4 * g) ^ (4 * (column & 7)))) = o[t];
  __syncthreads();
  constexpr int kParts = D / 4;
  const float value_scale = kE4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  for (int i = static_cast<int>(threadIdx.x); i < heads * kParts; i += kWaves * kWave) {
    const int c = i / kParts, d = 4 * (i % kParts);
    float highest = -__builtin_huge_valf();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, shared.stats[w][c].x);
    const float base = highest == -__builtin_huge_valf() ? 0.0f : highest;
    float total = 0.0f;
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 stat = shared.stats[w][c];
      const float weight = exp2_fast(stat.x - base);
      total += weight * stat.y;
      const floatx4 part = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(shared.values[w]) + c * D + (d ^ (4 * (c & 7))));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmaf(weight, part[k], v[k]);
    }
    if (u.splits > 1) {
      const int64_t at = (static_cast<int64_t>(u.part) * a.kv_heads + head) * 16 + c;
      *reinterpret_cast<floatx4*>(a.single_sums + at * D + d) = v;
      if (d == 0) a.single_stats[at] = make_float2(highest, total);
    } else {
      const bool nothing = highest == -__builtin_huge_valf();
      const float inverse = value_scale / total;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = nothing ? 0.0f : v[k] * inverse;
      store_row4(a.out + row * a.out_row + (q_head0 + c) * a.out_head + d, v);
    }
  }
}

// A workgroup's share of the single tokens' blocks: parts of one tile or of several.
template <int D, bool kE4m3, int kWaves>
__device__ __forceinline__ void decode_share(const PagedArgs& a, int workgroup, int head, DecodeShared<D, kWaves>& shared) {
  PagedShares shares;
  shares.start(a);
  const int64_t first = static_cast<int64_t>(workgroup) * shares.each;
  if (first >= shares.total) return;
  int at = static_cast<int>(first);
  const int end = static_cast<int>(min(first + shares.each, static_cast<int64_t>(shares.total)));
  for (;;) {
    PagedUnit u = shares.find(a, at);
    if (!u.live) return;
    const bool whole = u.from == 0 && u.blocks <= end - at;
    u.blocks = min(u.blocks, end - at);
    u.splits = whole ? 1 : 2;
    u.part = 2 * workgroup + (u.from == 0 ? 1 : 0);
    decode_unit<D, kE4m3, kWaves>(a, u, head, shared);
    at += u.blocks;
    if (at >= end) return;
    __syncthreads();  // (the rows in LDS have been read)
  }
}

}  // namespace d3
