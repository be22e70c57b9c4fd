// Attention of chunks of new tokens over a paged cache: tiles of 128 packed
// rows, one pass over the keys.
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
#include "paged_attention.h"

namespace d3 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kTileRows = 32 * kWaves;

// Byte of 16-byte part c of LDS row r: keys are read 16 rows at a time at one
// part, values in 32-byte pieces of 8 rows (D = 64: two rows share a bank row).
template <int D>
__device__ __forceinline__ int key_part(int r, int c) {
  return r * (2 * D) + ((c ^ (D >= 128 ? r & 15 : (r >> 1) & 7)) << 4);
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
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A word of two bf16 values with 0 in the place of an infinity or a NaN.
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

template <int D, bool kE4m3>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void paged_tile_kernel(PagedArgs a) {
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowParts = D * kBytes / 16;          // 16-byte parts of a cached row
  constexpr int kKeys = D == 256 ? 32 : 64;                 // of a step: what registers and LDS hold twice
  constexpr int kHalves = kKeys / 32;
  constexpr int kLoads = kKeys * kRowParts / kThreads;  // of keys, and of values, a thread
  constexpr int kKeysALoad = kThreads / kRowParts;
  constexpr int kSteps = D / 16, kColumns = D / 32;
  constexpr int kBlockBytes = kKeys * D * 2;
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t block[2][2][kBlockBytes];  // [buffer][keys, values], first: a load's place is 16 bits
    int infinite;                      // the last block whose values held an infinity or a NaN
  } shared;
  auto& lds = shared.block;
  int& infinite = shared.infinite;

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int column = lane & 31, half = lane >> 5;
  const int head = static_cast<int>(blockIdx.x) % a.kv_heads;
  if (a.zero_rest) paged_zero_rest(a, blockIdx.x, gridDim.x, D);
  const PagedUnit u = paged_unit<false>(a, static_cast<int>(blockIdx.x) / a.kv_heads);
  if (!u.live) return;

  const int all_rows = u.tokens * a.group;  // packed rows of the sequence
  const int tile_row = u.tile * kTileRows;
  const int last_row = min(tile_row + kTileRows, all_rows) - 1;
  const int before = u.length - u.tokens;
  const int64_t slot = paged_index(a.sequence_slots, a.slots_64, u.sequence);
  PagedKeys range = paged_keys(a, u, tile_row / a.group, last_row / a.group);
  if (slot < 0 || slot >= a.slots) range.high = range.low;
  const int32_t* pages = a.page_table + (slot < 0 || slot >= a.slots ? 0 : slot) * a.table_stride;
  const uint8_t* keys = a.keys + head * a.k_head;
  const uint8_t* values = a.values + head * a.v_head;
  const int in_page = (1 << a.page_shift) - 1;
  const float key_scale = a.scale * (kE4m3 && a.k_scales != nullptr ? a.k_scales[head] : 1.0f);

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
      qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const RowVector4*>(q + 16 * s));
  }

  floatx16 o[kColumns];
#pragma unroll
  for (int t = 0; t < kColumns; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
  float top = -__builtin_huge_valf(), sum = 0.0f;

  // Row of a transposing read, and the 16-byte part (its row's turn repeats every 8 rows).
  const int value_row = 4 * half + ((lane & 15) >> 2), value_column = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);

  // Staging.  bf16 blocks go from memory to LDS without registers: load i of wave w
  // fills 1 KiB, a lane's 16 bytes at their swizzled place by reading the part that
  // belongs there.  e4m3 ones are widened on the way.
  constexpr int kParts = kE4m3 ? kRowParts : D / 8;  // (of an LDS row, where the loads go by that)
  int32x4 kr[kE4m3 ? kLoads : 1], vr[kE4m3 ? kLoads : 1];
  auto page_of = [&](int key) -> int {  // of the block's key `lane`, -1 where nothing is attended
    const int at = key + (lane & (kKeys - 1));
    const bool in = at >= range.low && at < range.high;
    const int page = pages[in ? at >> a.page_shift : 0];
    return in && static_cast<uint32_t>(page) < a.pages ? page : -1;
  };
  auto load_block = [&](int key, int page, int buffer) {
    int thread = tid;
    asm volatile("" : "+v"(thread));  // (its places are worked out anew, not held in registers)
    const int my_part = thread % kParts, my_key = thread / kParts;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = my_key + i * kKeysALoad;
      const int p = __shfl(page, r, kWave);
      const int64_t token = (key + r) & in_page;
      const uint8_t* k = keys + p * a.k_page + token * a.k_token;
      const uint8_t* v = values + p * a.v_page + token * a.v_token;
      if (p < 0) k = paged_nothing, v = paged_nothing;
      if constexpr (kE4m3) {
        kr[i] = *reinterpret_cast<const int32x4*>(k + 16 * my_part);
        vr[i] = *reinterpret_cast<const int32x4*>(v + 16 * my_part);
      } else {  // (the part stored at place c of row r is c ^ the row's turn)
        const int at = (i * kWaves + wave) * 1024;
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
    for (int i = 0; i < kBlockBytes / (16 * kThreads); ++i) {
      int32x4* at = reinterpret_cast<int32x4*>(v + 16 * (i * kThreads + tid));
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
      const bool attends = key + c <= position && key + c > oldest;
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
            const uint32_t rest = attends ? w[j] ^ finite_of(w[j]) : 0u;  // only the infinities and NaN
            o[t][4 * i + 2 * j] += bf16_lo(rest);
            o[t][4 * i + 2 * j + 1] += bf16_hi(rest);
          }
        }
    }
  };

  int key = range.low & ~(kKeys - 1);
  int here = page_of(key);  // pages of this block's keys, and of the next one's
  uint64_t attended = __ballot(here >= 0);
  if (tid == 0) infinite = -1;
  if (key < range.high) {
    load_block(key, here, 0);
    store_block(0);
  }
  int page = page_of(key + kKeys);
  const int tile_low = before + tile_row / a.group, tile_oldest = behind(before + last_row / a.group);
  __syncthreads();
  for (int buffer = 0; key < range.high; buffer ^= 1, key += kKeys) {
    const bool more = key + kKeys < range.high;
    if (more) load_block(key + kKeys, page, buffer ^ 1);
    const int further = page_of(key + 2 * kKeys);
    if (key + kKeys - 1 > tile_low || key <= tile_oldest) {
      zero_infinite(key, lds[buffer][1]);
      lds_barrier();
    }
    // Blocks that no row of the wave attends are only staged.
    const bool mine = wave_live && key <= wave_high && key + kKeys - 1 > oldest_low;
    if (mine) {
      const uint8_t *k = lds[buffer][0], *v = lds[buffer][1];
      // Parts of a row differ by an exclusive or of the lane's own: one instruction a
      // read, where addresses held in registers would cost the kernel its second wave.
      int key_at = key_part<D>(column, half), value_at = value_part<D>(value_row, value_column) + 8 * (lane & 1);
      asm volatile("" : "+v"(key_at), "+v"(value_at));
      floatx16 s[kHalves];
#pragma unroll
      for (int b = 0; b < kHalves; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const bf16x8 w = *reinterpret_cast<const bf16x8*>(k + (key_at ^ (32 * st)) + 32 * b * (2 * D));
          s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, qf[st], s[b], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int b = 0; b < kHalves; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] *= key_scale;
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
      auto attends = [&](int b, int i) { return ((b ? mask_hi : mask_lo) >> (8 * (i >> 2) + (i & 3)) & 1u) != 0; };
      if (uneven || attended != ~uint64_t{0}) {
#pragma unroll
        for (int b = 0; b < kHalves; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] = attends(b, i) ? s[b][i] : -__builtin_huge_valf();
      }
      float most = s[0][0];
#pragma unroll
      for (int b = 0; b < kHalves; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[b][i]);
      most = max_across_32(most);
      if (__any(most > top)) {
        const float higher = fmaxf(top, most);
        const float shrink = top == higher ? 1.0f : exp2_fast(top - higher);
        top = higher;
        sum *= shrink;
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
          s[b][i] = exp2_fast(s[b][i] - base);
          sum += s[b][i];
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
      for (int e = 0; e < 2 * kHalves; ++e)
#pragma unroll
        for (int t = 0; t < kColumns; ++t) {
          uint32_t w[4];
          value_operand(t, e, w);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(w[0], w[1], w[2], w[3]), p[e], o[t], 0, 0, 0);
        }
      if (uneven && infinite == key) add_infinite(key, here);
    }
    if (more) store_block(buffer ^ 1);
    here = page, page = further;
    attended = __ballot(here >= 0);
    __syncthreads();
  }

  sum = sum_across_32(sum);
  if (!wave_live || wave_row + column > last_row) return;
  if (u.splits > 1) {
    const int64_t at = (static_cast<int64_t>(u.partial + u.split) * a.kv_heads + head) * kTileRows + 32 * wave + column;
#pragma unroll
    for (int t = 0; t < kColumns; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(a.sums + at * D + 32 * t + 8 * i + 4 * half) =
            floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    if (half == 0) a.stats[at] = make_float2(top, sum);
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

// Adds the splits of a tile's rows at the weights of their maxima, in split
// order; 16 rows a workgroup.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedArgs a, int parts, int row_parts, bool e4m3) {
  const int part = static_cast<int>(blockIdx.x) % parts;  // kv head and 16 rows of the tile
  const int head = part / row_parts, row16 = part % row_parts;
  const PagedUnit u = paged_unit<true>(a, static_cast<int>(blockIdx.x) / parts);
  if (!u.live) return;
  const int stored = a.tile_rows ? a.tile_rows : 16;
  const float value_scale = e4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  constexpr int kParts = D / 4;
  for (int i = static_cast<int>(threadIdx.x); i < 16 * kParts; i += kThreads) {
    const int r = 16 * row16 + i / kParts, d = 4 * (i % kParts);
    int token, member;
    if (a.tile_rows) {
      const int m = u.tile * a.tile_rows + r;
      if (m >= u.tokens * a.group) continue;
      token = m / a.group, member = m - token * a.group;
    } else {
      token = u.tile / a.slices, member = 16 * (u.tile % a.slices) + r;
      if (member >= a.group) continue;
    }
    const int64_t at = (static_cast<int64_t>(u.partial) * a.kv_heads + head) * stored + r;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * stored;
    float highest = -__builtin_huge_valf();
    for (int s = 0; s < u.splits; ++s) highest = fmaxf(highest, a.stats[at + s * step].x);
    const float base = highest == -__builtin_huge_valf() ? 0.0f : highest;
    float total = 0.0f;
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < u.splits; ++s) {
      const float2 stat = a.stats[at + s * step];
      const floatx4 w = *reinterpret_cast<const floatx4*>(a.sums + (at + s * step) * D + d);
      const float weight = exp2_fast(stat.x - base);
      total += weight * stat.y;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmaf(weight, w[k], v[k]);
    }
    const float inverse = total == 0.0f ? 0.0f : value_scale / total;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : v[k] * inverse;
    store_row4(a.out + static_cast<int64_t>(u.first_row + token) * a.out_row + (head * a.group + member) * a.out_head + d, v);
  }
}

// How a call is cut: decided by sizes the host knows.
constexpr int kCus = 256;

struct PagedPlan {
  bool decode;
  int slices, tile_rows, tile_tokens, target, least;
  int64_t max_units;
  bool split;  // whether a sequence can be long enough to be split
  int64_t partials;
};

PagedPlan paged_plan(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences, int32_t max_length) {
  PagedPlan p;
  const int64_t group = q_heads / c->kv_heads;
  p.decode = max_length <= 1;
  p.slices = static_cast<int>((group + 15) / 16);
  p.tile_rows = p.decode ? 0 : kTileRows;
  p.tile_tokens = p.decode ? 1 : static_cast<int>(kTileRows / group + 2);
  const int64_t tiles =
      p.decode ? rows * p.slices : rows * group / kTileRows + (sequences < rows ? sequences : rows);
  p.target = 2 * kCus / c->kv_heads > 0 ? 2 * kCus / c->kv_heads : 1;
  p.least = p.decode ? 2 : 4;
  const int64_t blocks = (static_cast<int64_t>(c->max_pages) * c->page_size + kKeyBlock - 1) / kKeyBlock;
  p.split = blocks > p.least && sequences > 0;
  p.max_units = tiles + (p.split ? p.target : 0);
  if (p.max_units < 1) p.max_units = 1;  // (no sequences: rows to zero)
  p.partials = p.split ? 2 * static_cast<int64_t>(p.target) : 0;
  return p;
}

int64_t sum_floats(const PagedPlan& p, const d3_paged_cache* c) {
  return p.partials * c->kv_heads * (p.tile_rows ? p.tile_rows : 16) * c->head_dim;
}

bool attention_suited(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences) {
  return (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && rows * q_heads <= (int64_t{1} << 23) &&
         sequences <= 65536;
}

}  // namespace

void launch_paged_tiles(const PagedArgs& a, int head_dim, bool e4m3, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.max_units) * a.kv_heads), block(kThreads);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  if (head_dim == 64)
    e4m3 ? run(paged_tile_kernel<64, true>) : run(paged_tile_kernel<64, false>);
  else if (head_dim == 128)
    e4m3 ? run(paged_tile_kernel<128, true>) : run(paged_tile_kernel<128, false>);
  else
    e4m3 ? run(paged_tile_kernel<256, true>) : run(paged_tile_kernel<256, false>);
}

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
  return sum_floats(p, cache) / cache->head_dim * (cache->head_dim + 2) * 4;
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
  const int64_t floats = sum_floats(p, cache);
  D3_REQUIRE(floats == 0 || (workspace && aligned_to(workspace, 16) &&
                             workspace_bytes >= floats / cache->head_dim * (cache->head_dim + 2) * 4),
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
  a.slices = p.slices, a.tile_rows = p.tile_rows, a.tile_tokens = p.tile_tokens;
  a.scale = scale * 1.4426950408889634f;
  a.window = static_cast<int>(window < 0 ? 0 : (window < 0x7fffffff ? window : 0x7fffffff));
  a.target = p.target, a.least = p.split ? p.least : 1 << 30;
  a.max_units = static_cast<int>(p.max_units);
  a.zero_rest = zero_rest;
  a.sums = static_cast<float*>(workspace);
  a.stats = floats ? reinterpret_cast<float2*>(a.sums + floats) : nullptr;
  if (p.decode)
    launch_paged_decode(a, cache->head_dim, e4m3, as_stream(stream));
  else
    launch_paged_tiles(a, cache->head_dim, e4m3, as_stream(stream));
  if (p.split) {
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess)
      return set_error(D3_ERR_HIP, "paged_attention launch failed: %s", hipGetErrorString(status));
    const int row_parts = p.decode ? 1 : kTileRows / 16;
    const int parts = cache->kv_heads * row_parts;
    const int64_t tiles = p.max_units - p.target < p.target ? p.max_units - p.target : p.target;
    const dim3 grid(static_cast<unsigned>(tiles * parts)), block(kThreads);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), a, parts, row_parts, e4m3); };
    if (cache->head_dim == 64)
      run(paged_join_kernel<64>);
    else if (cache->head_dim == 128)
      run(paged_join_kernel<128>);
    else
      run(paged_join_kernel<256>);
  }
  D3_LAUNCHED("paged_attention");
}
