// Attention of chunks of new tokens over a paged cache: tiles of 128 packed
// rows, one pass over the keys; a sequence's single token among them as
// paged_decode.h takes it.
//
// Wave w of a workgroup holds rows 32 w .. + 32 of the tile as columns of
// mfma_f32_32x32x16_bf16 and multiplies them with the workgroup's key block (64
// keys, staged in LDS): S^T = K Q^T, the running softmax in each lane's own
// column, O^T = V^T P^T with P^T as it lies in registers (keys numbered 8 (j / 4)
// + 4 h + j % 4 for lane half h, element j, in both operands).  Values are read
// from LDS transposed.
//
// Bound by the matrix cores and, as much, by the exponentials and the LDS reads:
// a wave reads every key and value of the block for its 32 rows.
#ifdef D3_TUNE
#include <stdlib.h>
#endif
#include "paged_decode.h"

namespace d3 {
namespace {

// Byte of 16-byte part c of LDS row r: keys are read 16 rows at a time at one
// part, values in 32-byte pieces of 8 rows (D = 64: two rows share a bank row).
template <int D>
__device__ __forceinline__ int key_part(int r, int c) {
  return r * (2 * D) + ((c ^ (D == 256 ? r & 7 : (D == 128 ? r & 15 : (r >> 1) & 7))) << 4);
}
template <int D>
__device__ __forceinline__ int value_part(int r, int c) {
  return r * (2 * D) + ((c ^ (2 * (D >= 128 ? r & 7 : (r >> 1) & 3))) << 4);
}

typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));

// 16 bytes a lane from memory to LDS at `to` + 16 * lane (`to` of the wave, the
// same in every lane).  As an instruction of its own: the compiler would wait for
// it at the next LDS read of any buffer.  wait_loads() and a barrier come before
// the first read of what it writes.  (m0 has no other use in the kernel.)
__device__ __forceinline__ void load_to_lds(const uint8_t* from, const uint8_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      static_cast<int>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)to)));
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from));
}
// The same from a wave's address and a lane's offset.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint32_t offset, const uint8_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      static_cast<int>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)to)));
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(from));
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A word of two bf16 values with 0 in the place of an infinity or a NaN.
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

constexpr int tile_keys(int dim) { return dim == 256 ? 32 : 64; }  // of a step: what registers and LDS hold twice

template <int D>
struct TileShared {
  // [buffer][keys, values], first: a load's place is 16 bits
  __attribute__((aligned(16))) uint8_t block[2][2][tile_keys(D) * D * 2];
  int infinite;  // the last block whose values held an infinity or a NaN
};

template <int D, bool kE4m3>
__device__ __forceinline__ void tile_unit(const PagedArgs& a, const PagedUnit& u, int head, TileShared<D>& shared) {
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowParts = D * kBytes / 16;  // 16-byte parts of a cached row
  constexpr int kKeys = tile_keys(D);
  constexpr int kHalves = kKeys / 32;
  constexpr int kLoads = kKeys * kRowParts / kPagedThreads;  // of keys, and of values, a thread
  constexpr int kKeysALoad = kPagedThreads / kRowParts;
  constexpr int kSteps = D / 16, kColumns = D / 32;
  constexpr int kBlockBytes = kKeys * D * 2;
  auto& lds = shared.block;
  int& infinite = shared.infinite;

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int column = lane & 31, half = lane >> 5;
  const int all_rows = u.tokens * a.group;  // packed rows of the sequence
  const int tile_row = u.tile * kTileRows;
  const int last_row = min(tile_row + kTileRows, all_rows) - 1;
  const int before = u.length - u.tokens;
  const PagedReach reach = paged_reach(a, u, tile_row / a.group, last_row / a.group, 6);
  const int blocks_each = ((reach.end - reach.aligned + kKeyBlock - 1) / kKeyBlock + u.splits - 1) / u.splits;
  const PagedKeys range = paged_keys(reach, u.split * blocks_each, blocks_each, 6);
  const int32_t* pages = a.page_table + (u.slot < 0 ? 0 : u.slot) * a.table_stride;
  const uint8_t* keys = a.keys + head * a.k_head;
  const uint8_t* values = a.values + head * a.v_head;
  const int in_page = (1 << a.page_shift) - 1;
  const ScoreScale scale = score_scale(a.scale * (kE4m3 && a.k_scales != nullptr ? a.k_scales[head] : 1.0f));

  // This lane's row, and the positions of the wave's.
  const int wave_row = tile_row + 32 * wave;
  const bool wave_live = wave_row <= last_row;
  const int my_row = min(wave_row + column, last_row);
  const int my_token = my_row / a.group;
  const int my_head = head * a.group + my_row - my_token * a.group;
  const int position = before + my_token;
  const int wave_low = before + min(wave_row, last_row) / a.group;
  const int wave_high = before + min(wave_row + 31, last_row) / a.group;
  // Keys up to these are out of the windows of this lane's row, the wave's first and its last.
  auto behind = [&](int p) { return a.window > 0 ? static_cast<int>(max(static_cast<int64_t>(p) - a.window, int64_t{-1})) : -1; };
  const int oldest = behind(position), oldest_low = behind(wave_low), oldest_high = behind(wave_high);
  bf16x8 qf[kSteps];
  {
    const uint16_t* q = a.q + static_cast<int64_t>(u.first_row + my_token) * a.q_row + my_head * a.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qf[s] = load_query(q + 16 * s, scale.sign);
  }

  floatx16 o[kColumns];
#pragma unroll
  for (int t = 0; t < kColumns; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
  // The weights' sums are one more row of values, all ones: the matrix cores have time
  // to spare, the vector units none.
  floatx16 sums;
#pragma unroll
  for (int i = 0; i < 16; ++i) sums[i] = 0.0f;
  const bf16x8 ones = operand(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  float top = -__builtin_huge_valf();

  // Row of a transposing read, and the 16-byte part (its row's turn repeats every 8 rows).
  const int value_row = 4 * half + ((lane & 15) >> 2), value_column = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);

  // Staging.  bf16 blocks go from memory to LDS without registers: load i of wave w
  // fills 1 KiB, a lane's 16 bytes at their swizzled place by reading the part that
  // belongs there.  e4m3 ones are widened on the way.
  constexpr int kParts = kE4m3 ? kRowParts : D / 8;  // (of an LDS row, where the loads go by that)
  int32x4 kr[kE4m3 ? kLoads : 1], vr[kE4m3 ? kLoads : 1];
  // The page of a block's key `lane`: the table's entry, loaded a block before it is
  // looked at (a use waits for every load before it); then -1 where nothing is attended.
  auto attends = [&](int key) { return key + (lane & (kKeys - 1)) >= range.low && key + (lane & (kKeys - 1)) < range.high; };
  auto entry_of = [&](int key) { return pages[attends(key) ? (key + (lane & (kKeys - 1))) >> a.page_shift : 0]; };
  auto page_of = [&](int key, int entry) { return attends(key) && static_cast<uint32_t>(entry) < a.pages ? entry : -1; };
  // A load's rows of one page, all attended: its address is the same for the wave but
  // for the lane's place, which no load changes (kKeysALoad rows turn alike).
  constexpr int kWaveRows = kWave / kRowParts;
  const bool by_page = !kE4m3 && (1 << a.page_shift) >= kWaveRows && max(a.k_token, a.v_token) < 1 << 24;
  const uint32_t lane_row = lane / kRowParts, lane_part = lane % kRowParts;
  const uint32_t k_lane = static_cast<uint32_t>(lane_row * a.k_token) + key_part<D>(kWaveRows * wave + lane_row, lane_part) - (kWaveRows * wave + lane_row) * 2 * D;
  const uint32_t v_lane = static_cast<uint32_t>(lane_row * a.v_token) + value_part<D>(kWaveRows * wave + lane_row, lane_part) - (kWaveRows * wave + lane_row) * 2 * D;
  // Where the rows of a block's keys begin: a lane's own key, so that the 64-bit
  // products are made once a block and a load reads its address from a lane.
  struct Rows {
    const uint8_t *key, *value;
  };
  auto rows_of = [&](int key, int page) {
    const int64_t token = (key + (lane & (kKeys - 1))) & in_page;
    Rows r;
    r.key = page < 0 ? paged_nothing : keys + page * a.k_page + token * a.k_token;
    r.value = page < 0 ? paged_nothing : values + page * a.v_page + token * a.v_token;
    return r;
  };
  // Load `piece` of a block whose loads go by pages: those of keys, then those of values.
  auto load_piece = [&](const Rows& rows, int buffer, int piece) {
    const int i = piece % kLoads, which = piece / kLoads;
    load_to_lds(lane_address(which ? rows.value : rows.key, i * kKeysALoad + kWaveRows * wave), which ? v_lane : k_lane,
                lds[buffer][which] + (i * kPagedWaves + wave) * 1024);
  };
  auto load_block = [&](const Rows& rows, int buffer) {
    int thread = tid;
    asm volatile("" : "+v"(thread));  // (its places are worked out anew, not held in registers)
    const int my_part = thread % kParts, my_key = thread / kParts;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = my_key + i * kKeysALoad;
      const uint8_t *k = shuffled_address(rows.key, r), *v = shuffled_address(rows.value, r);
      if constexpr (kE4m3) {
        kr[i] = *reinterpret_cast<const int32x4*>(k + 16 * my_part);
        vr[i] = *reinterpret_cast<const int32x4*>(v + 16 * my_part);
      } else {  // (the part stored at place c of row r is c ^ the row's turn)
        const int at = (i * kPagedWaves + wave) * 1024;
        load_to_lds(k + (key_part<D>(r, my_part) - r * (2 * D)), lds[buffer][0] + at);
        load_to_lds(v + (value_part<D>(r, my_part) - r * (2 * D)), lds[buffer][1] + at);
      }
    }
  };
  auto store_block = [&](int buffer) {
    if constexpr (kE4m3) {
      int thread = tid;
      asm volatile("" : "+v"(thread));
      const int my_part = thread % kParts, my_key = thread / kParts;
      uint8_t *k = lds[buffer][0], *v = lds[buffer][1];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = my_key + i * kKeysALoad;
        *reinterpret_cast<bf16x8*>(k + key_part<D>(r, 2 * my_part)) = widen8(kr[i][0], kr[i][1]);
        *reinterpret_cast<bf16x8*>(k + key_part<D>(r, 2 * my_part + 1)) = widen8(kr[i][2], kr[i][3]);
        *reinterpret_cast<bf16x8*>(v + value_part<D>(r, 2 * my_part)) = widen8(vr[i][0], vr[i][1]);
        *reinterpret_cast<bf16x8*>(v + value_part<D>(r, 2 * my_part + 1)) = widen8(vr[i][2], vr[i][3]);
      }
    } else {
      wait_loads();
    }
  };

  // Where the rows of a block's tile do not all attend the same of its keys, a row must
  // take nothing of a value that it does not attend, and 0 times an infinity or a NaN
  // is NaN: such blocks are searched for them, zeros put in their place for the
  // product, and what rows do attend added after it.
  auto zero_infinite = [&](int key, uint8_t* v) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < kBlockBytes / (16 * kPagedThreads); ++i) {
      int32x4* at = reinterpret_cast<int32x4*>(v + 16 * (i * kPagedThreads + tid));
      const int32x4 w = *at;
      int32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = static_cast<int>(finite_of(w[j]));
      if (f[0] != w[0] || f[1] != w[1] || f[2] != w[2] || f[3] != w[3]) *at = f, found = true;
    }
    if (found) infinite = key;
  };
  auto add_infinite = [&](int key, int page) {
#pragma unroll 1
    for (int c = 0; c < kKeys; ++c) {
      const int p = __shfl(page, c, kWave);
      if (p < 0) continue;
      const bool mine = key + c <= position && key + c > oldest;
      const uint8_t* row = values + p * a.v_page + ((key + c) & in_page) * a.v_token + 4 * kBytes * half;
#pragma unroll
      for (int t = 0; t < kColumns; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[2];
          if constexpr (kE4m3) {
            const bf16x8 wide = widen8(*reinterpret_cast<const uint32_t*>(row + 32 * t + 8 * i), 0);
            const int32x4 words = __builtin_bit_cast(int32x4, wide);
            w[0] = words[0], w[1] = words[1];
          } else {
            w[0] = *reinterpret_cast<const uint32_t*>(row + 64 * t + 16 * i);
            w[1] = *reinterpret_cast<const uint32_t*>(row + 64 * t + 16 * i + 4);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t rest = mine ? w[j] ^ finite_of(w[j]) : 0u;  // only the infinities and NaN
            o[t][4 * i + 2 * j] += bf16_lo(rest);
            o[t][4 * i + 2 * j + 1] += bf16_hi(rest);
          }
        }
    }
  };

  int key = range.low & ~(kKeys - 1);
  int here = page_of(key, entry_of(key));  // pages of this block's keys
  uint64_t attended = __ballot(here >= 0);
  if (tid == 0) infinite = -1;
  if (key < range.high) {
    load_block(rows_of(key, here), 0);
    store_block(0);
  }
  int entry = entry_of(key + kKeys);
  const int tile_low = before + tile_row / a.group, tile_oldest = behind(before + last_row / a.group);
  __syncthreads();
  for (int buffer = 0; key < range.high; buffer ^= 1, key += kKeys) {
    const bool more = key + kKeys < range.high;
    const int page = page_of(key + kKeys, entry);
    const uint64_t next_attended = __ballot(page >= 0);
    entry = entry_of(key + 2 * kKeys);
    // Loads wait for one another: those of a whole block go among the products.
    const bool pieces = !kE4m3 && more && by_page && next_attended == ~uint64_t{0};
    const Rows rows = rows_of(key + kKeys, page);
    if (more && !pieces) load_block(rows, buffer ^ 1);
    if (key + kKeys - 1 > tile_low || key <= tile_oldest) {
      zero_infinite(key, lds[buffer][1]);
      lds_barrier();
    }
    // Blocks that no row of the wave attends are only staged.
    const bool mine = wave_live && key <= wave_high && key + kKeys - 1 > oldest_low;
    if (!mine && pieces) {
#pragma unroll
      for (int i = 0; i < 2 * kLoads; ++i) load_piece(rows, buffer ^ 1, i);
    }
    if (mine) {
      const uint8_t *k = lds[buffer][0], *v = lds[buffer][1];
      // Parts of a row differ by an exclusive or of the lane's own: one instruction a
      // read, where addresses held in registers would cost the kernel its second wave.
      int key_at = key_part<D>(column, half), value_at = value_part<D>(value_row, value_column) + 8 * (lane & 1);
      asm volatile("" : "+v"(key_at), "+v"(value_at));
      floatx16 s[kHalves];
      auto scores = [&](auto with_loads) {
        constexpr int kEvery = kHalves * kSteps / (2 * kLoads);  // products a piece
#pragma unroll
        for (int b = 0; b < kHalves; ++b) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            const bf16x8 w = *reinterpret_cast<const bf16x8*>(k + (key_at ^ (32 * st)) + 32 * b * (2 * D));
            s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, qf[st], s[b], 0, 0, 0);
            if constexpr (decltype(with_loads)::value)
              if ((b * kSteps + st) % kEvery == 0) load_piece(rows, buffer ^ 1, (b * kSteps + st) / kEvery);
          }
        }
      };
      if constexpr (kE4m3) {
        scores(std::false_type{});
      } else {
        if (pieces)
          scores(std::true_type{});
        else
          scores(std::false_type{});
      }
      __builtin_amdgcn_sched_barrier(0);
      // Rows of the wave attend different keys of the block, or none of some: bit c
      // of the lane's mask is key 4 half + c of the block.
      const bool uneven = key + kKeys - 1 > wave_low || key <= oldest_high;
      uint64_t mask = attended;
      if (uneven) {
        const int newest = position - key, stale = oldest - key + 1;  // bits above and below them go
        mask &= newest < 0 ? 0 : ~uint64_t{0} >> (newest < 63 ? 63 - newest : 0);
        mask &= stale <= 0 ? ~uint64_t{0} : (stale < 64 ? ~uint64_t{0} << stale : 0);
      }
      mask >>= 4 * half;
      uint32_t mask_lo = static_cast<uint32_t>(mask), mask_hi = static_cast<uint32_t>(mask >> 32);
      auto seen = [&](int b, int i) { return ((b ? mask_hi : mask_lo) >> (8 * (i >> 2) + (i & 3)) & 1u) != 0; };
      if (uneven || attended != ~uint64_t{0}) {
#pragma unroll
        for (int b = 0; b < kHalves; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] = seen(b, i) ? s[b][i] : -__builtin_huge_valf();
      }
      float most = s[0][0];
#pragma unroll
      for (int b = 0; b < kHalves; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[b][i]);
      most = max_across_32(most) * scale.size;
      if (__any(most > top)) {
        const float higher = fmaxf(top, most);
        const float shrink = top == higher ? 1.0f : exp2_fast(top - higher);
        top = higher;
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[i] *= shrink;
#pragma unroll
        for (int t = 0; t < kColumns; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t][i] *= shrink;
      }
      const float base = top == -__builtin_huge_valf() ? 0.0f : top;
      bf16x8 p[2 * kHalves];
#pragma unroll
      for (int b = 0; b < kHalves; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[b][i] = exp2_fast(fmaf(s[b][i], scale.size, -base));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          p[2 * b + e] = operand(pack_bf16x2(s[b][8 * e], s[b][8 * e + 1]), pack_bf16x2(s[b][8 * e + 2], s[b][8 * e + 3]),
                                 pack_bf16x2(s[b][8 * e + 4], s[b][8 * e + 5]), pack_bf16x2(s[b][8 * e + 6], s[b][8 * e + 7]));
      }
      auto value_operand = [&](int t, int step, uint32_t* w) {
        const uint8_t* at = v + (value_at ^ (64 * t)) + 16 * step * (2 * D);
        const uint32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * (2 * D));
        w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
      };
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 2 * kHalves; ++e) {
        sums = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ones, p[e], sums, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < kColumns; ++t) {
          uint32_t w[4];
          value_operand(t, e, w);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(w[0], w[1], w[2], w[3]), p[e], o[t], 0, 0, 0);
        }
      }
      if (uneven && infinite == key) add_infinite(key, here);
    }
    if (more) store_block(buffer ^ 1);
    here = page;
    attended = next_attended;
    __syncthreads();
  }

  const float sum = sums[0];
  if (!wave_live || wave_row + column > last_row) return;
  if (u.splits > 1) {
    const int64_t at = (static_cast<int64_t>(u.part) * a.kv_heads + head) * kTileRows + 32 * wave + column;
#pragma unroll
    for (int t = 0; t < kColumns; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(a.tile_sums + at * D + 32 * t + 8 * i + 4 * half) =
            floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    if (half == 0) a.tile_stats[at] = make_float2(top, sum);
    return;
  }
  const float value_scale = kE4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  const float inverse = sum == 0.0f ? 0.0f : value_scale / sum;
  uint16_t* out = a.out + static_cast<int64_t>(u.first_row + my_token) * a.out_row + my_head * a.out_head;
#pragma unroll
  for (int t = 0; t < kColumns; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      floatx4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = sum == 0.0f ? 0.0f : o[t][4 * i + j] * inverse;
      store_row4(out + 32 * t + 8 * i + 4 * half, w);
    }
}

template <int D, bool kE4m3>
__global__ __launch_bounds__(kPagedThreads, D == 256 ? 1 : 2) void paged_tile_kernel(PagedArgs a) {
  __shared__ union Shared {
    __device__ Shared() {}
    DecodeShared<D, kE4m3> decode;
    TileShared<D> tile;
  } shared;
  const int unit = static_cast<int>(blockIdx.x) / a.kv_heads, head = static_cast<int>(blockIdx.x) % a.kv_heads;
  if (unit < a.shares) {
    decode_share<D, kE4m3>(a, unit, head, shared.decode);
  } else if (unit < a.shares + a.tile_units) {
    const PagedUnit u = paged_tile_unit<false>(a, unit - a.shares);
    if (u.live) tile_unit<D, kE4m3>(a, u, head, shared.tile);
  } else {
    paged_zero_rest(a, static_cast<int>(blockIdx.x) - (a.tile_units + a.shares) * a.kv_heads, D);
  }
}

// Adds the parts of a tile's rows at the weights of their maxima, in the order of
// their keys; a thread takes four columns of one of 16 rows, eight parts in flight.
template <int D>
__global__ __launch_bounds__(4 * D) void paged_join_kernel(PagedArgs a, int tiles, bool e4m3) {
  constexpr int kBatch = 8;
  constexpr int kRowParts = kTileRows / 16;
  const int r = static_cast<int>(threadIdx.x) / (D / 4), d = 4 * (static_cast<int>(threadIdx.x) % (D / 4));
  PagedUnit u;
  int head, token, member;
  int64_t at, step;
  const float* sums;
  const float2* stats;
  if (static_cast<int>(blockIdx.x) < tiles * a.kv_heads * kRowParts) {
    const int part = static_cast<int>(blockIdx.x) % (a.kv_heads * kRowParts);
    head = part % a.kv_heads;
    u = paged_tile_unit<true>(a, static_cast<int>(blockIdx.x) / (a.kv_heads * kRowParts));
    if (!u.live) return;
    const int row = 16 * (part / a.kv_heads) + r, m = u.tile * kTileRows + row;
    if (m >= u.tokens * a.group) return;
    token = m / a.group, member = m - token * a.group;
    at = (static_cast<int64_t>(u.part) * a.kv_heads + head) * kTileRows + row, step = a.kv_heads * kTileRows;
    sums = a.tile_sums, stats = a.tile_stats;
  } else {
    // The tile that the share of workgroup w ends in, where it is the tile's first part.
    const int group = static_cast<int>(blockIdx.x) - tiles * a.kv_heads * kRowParts;
    const int w = group / a.kv_heads;
    head = group % a.kv_heads;
    PagedShares shares;
    shares.start(a);
    const int64_t end = static_cast<int64_t>(w + 1) * shares.each;
    if (end >= shares.total) return;
    u = shares.find(a, static_cast<int>(end));
    if (!u.live || u.from == 0 || u.from > shares.each) return;
    // (a share that began with the tile ends `each` into it, any other less)
    const int tile_end = u.from + u.blocks;  // blocks of the tile
    u.splits = 1 + (tile_end - u.from + shares.each - 1) / shares.each;
    u.part += w;
    if (u.part < 0 || u.part > a.single_parts - u.splits) return;
    token = u.tile / a.slices, member = 16 * (u.tile % a.slices) + r;
    if (member >= a.group) return;
    at = (static_cast<int64_t>(u.part) * a.kv_heads + head) * 16 + r, step = a.kv_heads * 16;
    sums = a.single_sums, stats = a.single_stats;
  }
  const float value_scale = e4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  float highest = -__builtin_huge_valf(), total = 0.0f;
  floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < u.splits; s += kBatch) {
    float2 stat[kBatch];
    floatx4 w[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t from = at + min(s + b, u.splits - 1) * step;
      stat[b] = stats[from];
      w[b] = *reinterpret_cast<const floatx4*>(sums + from * D + d);
    }
    float higher = highest;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) higher = fmaxf(higher, stat[b].x);
    const float base = higher == -__builtin_huge_valf() ? 0.0f : higher;
    const float shrink = highest == higher ? 1.0f : exp2_fast(highest - base);
    total *= shrink;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= shrink;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (s + b >= u.splits) break;
      const float weight = exp2_fast(stat[b].x - base);
      total += weight * stat[b].y;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmaf(weight, w[b][k], v[k]);
    }
    highest = higher;
  }
  const float inverse = total == 0.0f ? 0.0f : value_scale / total;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : v[k] * inverse;
  store_row4(a.out + static_cast<int64_t>(u.first_row + token) * a.out_row + (head * a.group + member) * a.out_head + d, v);
}

// How a call is cut, as far as the host knows its sizes.
constexpr int kCus = 256;

#ifdef D3_TUNE
int tuned(const char* name, int v) { const char* e = getenv(name); return e ? atoi(e) : v; }
#else
constexpr int tuned(const char*, int v) { return v; }
#endif

struct PagedPlan {
  bool all_single, split_tiles, split_shares;
  int slices, tile_tokens, share_shift, shares, least, target, least_split;
  int64_t tiles, tile_units, single_parts, tile_parts;
};

PagedPlan paged_plan(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences, int32_t max_length) {
  PagedPlan p = {};
  const int64_t group = q_heads / c->kv_heads;
  const int64_t capacity = static_cast<int64_t>(c->max_pages) * c->page_size;
  const int64_t some = sequences < rows ? sequences : rows;
  p.all_single = max_length <= 1;
  p.slices = static_cast<int>((group + 15) / 16);
  p.tile_tokens = p.all_single ? 1 : static_cast<int>(kTileRows / group + 2);
  // Single tokens: blocks of 64 keys; one block a tile where no slot holds more keys
  // than are worth a second launch; larger where all of them could be 2^30 and more.
  const int64_t single_tiles = (p.all_single ? rows : some) * p.slices;
  p.share_shift = 6;
  while (capacity <= tuned("D3_ALONE", 512) && capacity > 1 << p.share_shift) ++p.share_shift;
  while ((((capacity - 1) >> p.share_shift) + 1) * single_tiles >= int64_t{1} << 30) ++p.share_shift;
  const int64_t blocks = ((capacity - 1) >> p.share_shift) + 1;
  const int resident = (p.all_single ? tuned("D3_PER_CU", c->head_dim == 64 ? 4 : 2) : tuned("D3_MIXED", 1)) * kCus / c->kv_heads;
  p.least = blocks > 1 ? tuned("D3_LEAST", 4) : 1;
  // No more workgroups than the blocks can give work to.
  const int64_t useful = (single_tiles * blocks + p.least - 1) / p.least;
  p.shares = sequences == 0 ? 0 : static_cast<int>(useful < resident ? useful : (resident > 0 ? resident : 1));
  p.split_shares = p.shares > 1 && blocks > 1;
  p.single_parts = p.split_shares ? p.shares + single_tiles : 0;
  // Tiles of more rows.
  p.target = tuned("D3_TARGET", 2) * kCus / c->kv_heads;
  if (p.target < 1) p.target = 1;
  p.least_split = tuned("D3_SPLIT", 8);
  if (!p.all_single && sequences > 0) {
    p.tiles = rows * group / kTileRows + some;
    p.split_tiles = (capacity + kKeyBlock - 1) / kKeyBlock > p.least_split;
    p.tile_units = p.tiles + (p.split_tiles ? p.target : 0);
    p.tile_parts = p.split_tiles ? 2 * static_cast<int64_t>(p.target) : 0;
  }
  return p;
}

int64_t workspace_rows(const PagedPlan& p, const d3_paged_cache* c) {
  return (p.single_parts * 16 + p.tile_parts * kTileRows) * c->kv_heads;
}

bool attention_suited(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences) {
  return (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && rows * q_heads <= (int64_t{1} << 23) &&
         sequences <= 65536;
}

void launch_paged_tiles(const PagedArgs& a, int head_dim, bool e4m3, bool zero_rest, hipStream_t stream) {
  const unsigned workgroups = paged_workgroups(a, zero_rest);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(kPagedThreads), 0, stream, a); };
  if (head_dim == 64)
    e4m3 ? run(paged_tile_kernel<64, true>) : run(paged_tile_kernel<64, false>);
  else if (head_dim == 128)
    e4m3 ? run(paged_tile_kernel<128, true>) : run(paged_tile_kernel<128, false>);
  else
    e4m3 ? run(paged_tile_kernel<256, true>) : run(paged_tile_kernel<256, false>);
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int64_t d3_paged_attention_workspace(const d3_paged_cache* cache, int64_t rows, int32_t q_heads,
                                                int32_t sequences, int32_t max_length) {
  if (check_paged_cache("paged_attention_workspace", cache)) return -1;
  if (rows < 0 || sequences < 0 || q_heads <= 0 || q_heads % cache->kv_heads != 0 ||
      !attention_suited(cache, rows, q_heads, sequences))
    return -1;
  clear_error();
  if (rows == 0) return 0;
  const PagedPlan p = paged_plan(cache, rows, q_heads, sequences, max_length);
  return workspace_rows(p, cache) * (cache->head_dim + 2) * 4;
}

extern "C" int d3_paged_attention(const d3_paged_cache* cache, const uint16_t* q, int64_t q_row_stride,
                                  int64_t q_head_stride, int64_t rows, int32_t q_heads, const int32_t* boundaries,
                                  const void* sequence_slots, int32_t sequence_slots_dtype, const void* lengths,
                                  int32_t lengths_dtype, int32_t sequences, int32_t max_length, float scale,
                                  int64_t window, uint16_t* out, int64_t out_row_stride, int64_t out_head_stride,
                                  int32_t zero_rest, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int status = check_paged_cache("paged_attention", cache)) return status;
  D3_REQUIRE(rows >= 0 && sequences >= 0, "paged_attention: shape");
  D3_REQUIRE(q_heads > 0 && q_heads % cache->kv_heads == 0, "paged_attention: %d query heads, %d kv heads", q_heads,
             cache->kv_heads);
  D3_REQUIRE((sequence_slots_dtype == D3_DTYPE_I32 || sequence_slots_dtype == D3_DTYPE_I64) &&
                 (lengths_dtype == D3_DTYPE_I32 || lengths_dtype == D3_DTYPE_I64),
             "paged_attention: slots and lengths must be int32 or int64");
  D3_SUPPORTED(attention_suited(cache, rows, q_heads, sequences),
               "paged_attention: head dim %d (64, 128 or 256), %lld rows of %d heads, %d sequences", cache->head_dim,
               static_cast<long long>(rows), q_heads, sequences);
  D3_REQUIRE(rows == 0 || (q && out), "paged_attention: null pointer");
  D3_REQUIRE(rows == 0 || sequences == 0 || (boundaries && sequence_slots && lengths), "paged_attention: null pointer");
  if (rows == 0 || (sequences == 0 && !zero_rest)) {
    clear_error();
    return D3_OK;
  }
  const PagedPlan p = paged_plan(cache, rows, q_heads, sequences, max_length);
  const int64_t stored = workspace_rows(p, cache);
  D3_REQUIRE(stored == 0 || (workspace && aligned_to(workspace, 16) &&
                             workspace_bytes >= stored * (cache->head_dim + 2) * 4),
             "paged_attention: workspace");
  const bool e4m3 = cache->dtype == D3_DTYPE_E4M3;
  const int64_t size = e4m3 ? 1 : 2;
  PagedArgs a = {};
  a.q = q, a.q_row = q_row_stride, a.q_head = q_head_stride;
  a.out = out, a.out_row = out_row_stride, a.out_head = out_head_stride;
  a.keys = static_cast<const uint8_t*>(cache->keys), a.values = static_cast<const uint8_t*>(cache->values);
  a.k_page = cache->key_page_stride * size, a.k_token = cache->key_token_stride * size;
  a.k_head = cache->key_head_stride * size;
  a.v_page = cache->value_page_stride * size, a.v_token = cache->value_token_stride * size;
  a.v_head = cache->value_head_stride * size;
  a.page_table = cache->page_table, a.table_stride = cache->table_stride;
  a.pages = static_cast<uint32_t>(cache->pages), a.slots = cache->slots;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(cache->page_size));
  a.capacity = cache->max_pages * cache->page_size;
  a.k_scales = cache->key_scales, a.v_scales = cache->value_scales;
  a.boundaries = boundaries;
  a.sequence_slots = sequence_slots, a.slots_64 = sequence_slots_dtype == D3_DTYPE_I64;
  a.lengths = lengths, a.lengths_64 = lengths_dtype == D3_DTYPE_I64;
  a.sequences = sequences, a.rows = static_cast<int>(rows);
  a.q_heads = q_heads, a.kv_heads = cache->kv_heads, a.group = q_heads / cache->kv_heads;
  a.slices = p.slices, a.all_single = p.all_single, a.tile_tokens = p.tile_tokens;
  a.scale = scale * 1.4426950408889634f;
  a.window = static_cast<int>(window < 0 ? 0 : (window < 0x7fffffff ? window : 0x7fffffff));
  a.share_shift = p.share_shift, a.shares = p.shares, a.least = p.least;
  a.target = p.target, a.least_split = p.split_tiles ? p.least_split : 1 << 30;
  a.tile_units = static_cast<int>(p.tile_units);
  a.single_parts = static_cast<int>(p.single_parts), a.tile_parts = static_cast<int>(p.tile_parts);
  const int64_t single_rows = p.single_parts * 16 * cache->kv_heads;
  a.single_sums = static_cast<float*>(workspace);
  a.tile_sums = a.single_sums + single_rows * cache->head_dim;
  a.single_stats = reinterpret_cast<float2*>(a.single_sums + stored * cache->head_dim);
  a.tile_stats = a.single_stats + single_rows;
  if (p.all_single)
    launch_paged_decode(a, cache->head_dim, e4m3, zero_rest != 0, as_stream(stream));
  else
    launch_paged_tiles(a, cache->head_dim, e4m3, zero_rest != 0, as_stream(stream));
  if (p.split_tiles || p.split_shares) {
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess)
      return set_error(D3_ERR_HIP, "paged_attention launch failed: %s", hipGetErrorString(status));
    const int tiles = p.split_tiles ? static_cast<int>(p.tiles < p.target ? p.tiles : p.target) : 0;
    const int ends = p.split_shares ? p.shares - 1 : 0;
    const dim3 grid(static_cast<unsigned>((tiles * (kTileRows / 16) + ends) * cache->kv_heads)), block(4 * cache->head_dim);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), a, tiles, e4m3); };
    if (cache->head_dim == 64)
      run(paged_join_kernel<64>);
    else if (cache->head_dim == 128)
      run(paged_join_kernel<128>);
    else
      run(paged_join_kernel<256>);
  }
  D3_LAUNCHED("paged_attention");
}
