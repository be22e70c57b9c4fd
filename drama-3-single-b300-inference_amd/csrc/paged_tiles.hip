// Attention of chunks of new tokens over a paged cache: tiles of packed rows, one
// pass over the keys; a sequence's single token among them as paged_decode.h takes it.
//
// Wave w of a workgroup holds rows 32 w .. + 32 of the tile as columns of
// mfma_f32_32x32x16_bf16 and multiplies them with the workgroup's key block (64
// keys, staged in LDS): S^T = K Q^T, the running softmax in each lane's own
// column, O^T = V^T P^T with P^T as it lies in registers (keys numbered 8 (j / 4)
// + 4 h + j % 4 for lane half h, element j, in both operands).  Values are read
// from LDS transposed.
//
// Bound by the matrix cores and, as much, by the vector units: a block is 32
// products of 32 cycles a wave (128 columns) and about as long in exponentials (four
// times an ordinary instruction's time) and what goes with them.  Two ways to keep both
// busy: two workgroups a CU of one group of four waves each (128 rows), or one of two
// groups (256 rows) whose waves share a SIMD and take turns by barriers: while one
// multiplies (values of the last block, keys of this one), the other computes weights.
// 4096 rows over 20480 keys of 128 columns 1375-1427 us by the card (1070-1110 TFLOP/s; a
// product of 8192^3 by the library 1390), a prompt of 8192 281 us; 4096 rows over 4096 keys
// 950 TFLOP/s, from e4m3 890 (a block is widened between its products and the barrier,
// where the other group waits), of 64 columns 630 (half the products a weight, and nothing of
// a wave's own beside its weights), of 256 500 (one wave a SIMD).
#include "paged_decode.h"

namespace d3 {
namespace {

// Byte of 16-byte part c of LDS row r: keys are read 16 rows at a time at one
// part, values in 64-byte pieces of 4 rows (D = 64: two rows share a bank row); no
// two of them lie on one bank (measured: no conflicts).
template <int D>
__device__ __forceinline__ int key_part(int r, int c) {
  return r * (2 * D) + ((c ^ (D == 256 ? r & 7 : (D == 128 ? r & 15 : (r >> 1) & 7))) << 4);
}
template <int D>
__device__ __forceinline__ int value_part(int r, int c) {
  return r * (2 * D) + ((c ^ (D >= 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1))) << 4);
}

typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));

// 16 bytes a lane from memory to LDS at `to` + 16 * lane (`to` of the wave, the
// same in every lane).  As an instruction of its own: the compiler would wait for
// it at the next LDS read of any buffer.  wait_loads() and a barrier come before
// the first read of what it writes.  One wait state lies between the write of m0, which
// has no other use in the kernel, and the load.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, const uint8_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      static_cast<int>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from));
}
// The same from a wave's address and a lane's offset.  The address comes out of a lane
// (v_readlane), and a load may read an SGPR that a vector instruction wrote five wait
// states later at the earliest, which the compiler does not see to in here: a scalar
// copy, which waits by itself, is one.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint32_t offset, const uint8_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      static_cast<int>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)to)));
  uint64_t address;
  asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
               : "=&s"(address)
               : "s"(at), "v"(offset), "s"(from));
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A word of two bf16 values with 0 in the place of an infinity or a NaN.
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

// What a row's weights are powers of two above need not be its highest score: it is
// raised where a score is 2^8 times above it, and weights and sums reach 2^8 times
// more.  (Raised at every new maximum, a prompt of
// 8192 304 us, a chunk of 4096 over 20480 1478: so 290 and 1440.)
constexpr float kSlack = 8.0f;

constexpr int tile_keys(int dim) { return dim == 256 ? 32 : 64; }  // of a block

// A score, or minus infinity where the bit of the mask is 0.
__device__ __forceinline__ float attended_or_nothing(float score, uint32_t mask, int bit) {
  const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(mask), bit, 1));
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, score) & keep) | (0xff800000u & ~keep));
}

template <int D, int kGroups>
struct TileShared {
  // A block's keys (and values) are loaded once the group that is last done with its
  // buffer's block: two blocks before it where groups take turns, one where there is one.
  static constexpr int kBytes = tile_keys(D) * D * 2;
  __attribute__((aligned(16))) uint8_t keys[kGroups + 1][kBytes];
  __attribute__((aligned(16))) uint8_t values[kGroups + 1][kBytes];
  int infinite[kGroups + 1];  // the last block of each buffer whose values held an infinity or a NaN
};

template <int D, bool kE4m3, int kGroups>
__device__ __forceinline__ void tile_unit(const PagedArgs& a, const PagedUnit& u, int head, TileShared<D, kGroups>& shared) {
  constexpr int kWaves = 4 * kGroups, kThreads = kWaves * kWave, kBuffers = kGroups + 1;
  constexpr int kTileRows = kGroupRows * kGroups;
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowParts = D * kBytes / 16;  // 16-byte parts of a cached row
  constexpr int kKeys = tile_keys(D), kHalves = kKeys / 32;
  constexpr int kParts = kKeys * kRowParts;                               // of a block's keys, and of its values
  constexpr int kLoads = kParts < kThreads ? 1 : kParts / kThreads;       // a thread
  constexpr int kKeysALoad = kThreads / kRowParts, kWaveRows = kWave / kRowParts;
  constexpr int kSteps = D / 16, kColumns = D / 32;
  // Fragments in flight from LDS, in the order written here (4096 rows over 20480 keys:
  // 1398 us, three 1407; eight 1475, and 1437 where the compiler orders them).
  constexpr int kAhead = 4;

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int column = lane & 31, half = lane >> 5;
  const bool second = kGroups == 2 && wave >= 4;
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

  // This lane's row, and the positions of the wave's and of the tile's.
  const int wave_row = tile_row + 32 * wave;
  const bool wave_live = wave_row <= last_row;
  const int my_row = min(wave_row + column, last_row);
  const int my_token = my_row / a.group;
  const int my_head = head * a.group + my_row - my_token * a.group;
  const int position = before + my_token;
  const int wave_low = before + min(wave_row, last_row) / a.group;
  const int wave_high = wave_live ? before + min(wave_row + 31, last_row) / a.group : -1;  // (-1: attends no block)
  const int tile_low = before + tile_row / a.group;
  // Keys up to these are out of the windows of this lane's row, the wave's first and
  // its last, and the tile's last.
  auto behind = [&](int p) { return a.window > 0 ? static_cast<int>(max(static_cast<int64_t>(p) - a.window, int64_t{-1})) : -1; };
  const int oldest = behind(position), oldest_low = behind(wave_low), oldest_high = behind(wave_high);
  const int tile_oldest = behind(before + last_row / a.group);
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
  float sum = 0.0f;

  // The page of a block's key `lane`: the table's entry, loaded a block before it is
  // looked at (a use waits for every load before it); then -1 where nothing is attended.
  auto attends = [&](int key) { return key + (lane & (kKeys - 1)) >= range.low && key + (lane & (kKeys - 1)) < range.high; };
  auto entry_of = [&](int key) { return pages[attends(key) ? (key + (lane & (kKeys - 1))) >> a.page_shift : 0]; };
  auto page_of = [&](int key, int entry) { return attends(key) && static_cast<uint32_t>(entry) < a.pages ? entry : -1; };
  // Where its row begins: the products are made once a block, loads take it from there.
  auto row_of = [&](const uint8_t* base, uint32_t page_bytes, uint32_t token_bytes, int key, int page) {
    const uint64_t token = (key + (lane & (kKeys - 1))) & in_page;
    return page < 0 ? paged_nothing : base + (static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_bytes + token * token_bytes);
  };

  // Staging.  bf16 blocks go from memory to LDS without registers: load i of wave w
  // fills 1 KiB, a lane's 16 bytes at their swizzled place by reading the part that
  // belongs there.  Where a load's rows are of one page and all attended, its address
  // is the wave's but for the lane's place, which no load changes (kKeysALoad rows turn
  // alike).  e4m3 blocks are widened on the way.
  const bool by_page = !kE4m3 && (1 << a.page_shift) >= kWaveRows && max(a.k_token, a.v_token) < 1u << 24;
  const bool loading = kWaveRows * wave < kKeys;
  const int piecewise = __builtin_amdgcn_readfirstlane(by_page && loading);  // (a scalar register, where a condition is two)
  const int lane_row = lane / kRowParts, lane_part = lane % kRowParts;
  const int wave_first = kWaveRows * wave;  // of the wave's first load
  const uint32_t k_lane = lane_row * a.k_token + key_part<D>(wave_first + lane_row, lane_part) - (wave_first + lane_row) * 2 * D;
  const uint32_t v_lane = lane_row * a.v_token + value_part<D>(wave_first + lane_row, lane_part) - (wave_first + lane_row) * 2 * D;
  int32x4 kr[kE4m3 ? kLoads : 1], vr[kE4m3 ? kLoads : 1];
  auto load_piece = [&](const uint8_t* rows, uint32_t lane_place, uint8_t* to, int i) {
    load_to_lds(lane_address(rows, i * kKeysALoad + wave_first), lane_place, to + (i * kWaves + wave) * 1024);
  };
  auto load_keys = [&](const uint8_t* rows, uint8_t* to) {
    if (!loading) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = wave_first + lane_row + i * kKeysALoad;
      const uint8_t* from = shuffled_address(rows, r);
      if constexpr (kE4m3)
        kr[i] = *reinterpret_cast<const int32x4*>(from + 16 * lane_part);
      else  // (the part stored at place c of row r is c ^ the row's turn)
        load_to_lds(from + (key_part<D>(r, lane_part) - r * (2 * D)), to + (i * kWaves + wave) * 1024);
    }
  };
  auto load_values = [&](const uint8_t* rows, uint8_t* to) {
    if (!loading) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = wave_first + lane_row + i * kKeysALoad;
      const uint8_t* from = shuffled_address(rows, r);
      if constexpr (kE4m3)
        vr[i] = *reinterpret_cast<const int32x4*>(from + 16 * lane_part);
      else
        load_to_lds(from + (value_part<D>(r, lane_part) - r * (2 * D)), to + (i * kWaves + wave) * 1024);
    }
  };
  auto store_keys = [&](uint8_t* to) {  // (e4m3)
    if (!loading) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = wave_first + lane_row + i * kKeysALoad;
      *reinterpret_cast<bf16x8*>(to + key_part<D>(r, 2 * lane_part)) = widen8(kr[i][0], kr[i][1]);
      *reinterpret_cast<bf16x8*>(to + key_part<D>(r, 2 * lane_part + 1)) = widen8(kr[i][2], kr[i][3]);
    }
  };
  auto store_values = [&](uint8_t* to) {
    if (!loading) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = wave_first + lane_row + i * kKeysALoad;
      *reinterpret_cast<bf16x8*>(to + value_part<D>(r, 2 * lane_part)) = widen8(vr[i][0], vr[i][1]);
      *reinterpret_cast<bf16x8*>(to + value_part<D>(r, 2 * lane_part + 1)) = widen8(vr[i][2], vr[i][3]);
    }
  };

  // Where the rows of a block's tile do not all attend the same of its keys, a row must
  // take nothing of a value that it does not attend, and 0 times an infinity or a NaN
  // is NaN: each wave searches what it loaded of such a block for them and puts zeros in
  // their place for the product; what rows do attend is added after it.
  auto tile_uneven = [&](int key) { return key + kKeys - 1 > tile_low || key <= tile_oldest; };
  auto zero_infinite = [&](int key, uint8_t* v, int* flag) {
    if (!loading) return;
    auto pieces_of = [&](auto visit) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if constexpr (kE4m3) {
          const int r = wave_first + lane_row + i * kKeysALoad;
          visit(v + value_part<D>(r, 2 * lane_part));
          visit(v + value_part<D>(r, 2 * lane_part + 1));
        } else {
          visit(v + (i * kWaves + wave) * 1024 + 16 * lane);
        }
      }
    };
    uint16x2 largest = {0, 0};  // (first only whether there is any: 16 windowed prompts 64 us without)
    pieces_of([&](const uint8_t* at) {
      const int32x4 w = *reinterpret_cast<const int32x4*>(at);
#pragma unroll
      for (int j = 0; j < 4; ++j) largest = __builtin_elementwise_max(largest, __builtin_bit_cast(uint16x2, w[j] & 0x7fff7fff));
    });
    if (max(largest.x, largest.y) < 0x7f80) return;
    pieces_of([&](uint8_t* at) {
      int32x4* place = reinterpret_cast<int32x4*>(at);
      const int32x4 w = *place;
      int32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = static_cast<int>(finite_of(w[j]));
      if (f[0] != w[0] || f[1] != w[1] || f[2] != w[2] || f[3] != w[3]) *place = f;
    });
    *flag = key;
  };
  auto add_infinite = [&](int key) {
    const int page = page_of(key, entry_of(key));
#pragma unroll 1
    for (int c = 0; c < kKeys; ++c) {
      const int p = __shfl(page, c, kWave);
      if (p < 0) continue;
      const bool mine = key + c <= position && key + c > oldest;
      const uint8_t* row = values + static_cast<uint64_t>(p) * a.v_page + static_cast<uint64_t>((key + c) & in_page) * a.v_token + 4 * kBytes * half;
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

  // Blocks of the unit; rows of the wave attend a block, or none does.
  const int key0 = range.low & ~(kKeys - 1);
  const int blocks = range.low < range.high ? (range.high - key0 + kKeys - 1) / kKeys : 0;
  auto wave_attends = [&](int key) { return key <= wave_high && key + kKeys - 1 > oldest_low; };
  auto wave_uneven = [&](int key) { return key + kKeys - 1 > wave_low || key <= oldest_high; };

  // Before the first: its keys and values and the second's keys.
  int page1 = -1;  // of the next block's keys
  int entry = 0;   // table's, of the one after
  uint64_t attended = 0, attended1 = 0;
  if (blocks > 0) {
    const int page0 = page_of(key0, entry_of(key0));
    page1 = page_of(key0 + kKeys, entry_of(key0 + kKeys));
    entry = entry_of(key0 + 2 * kKeys);
    attended = __ballot(page0 >= 0), attended1 = __ballot(page1 >= 0);
    load_keys(row_of(keys, a.k_page, a.k_token, key0, page0), shared.keys[0]);
    load_values(row_of(values, a.v_page, a.v_token, key0, page0), shared.values[0]);
    if constexpr (kE4m3) store_keys(shared.keys[0]), store_values(shared.values[0]);
    load_keys(row_of(keys, a.k_page, a.k_token, key0 + kKeys, page1), shared.keys[1]);
    if constexpr (kE4m3) store_keys(shared.keys[1]);
    wait_loads();
    if (tid < kBuffers) shared.infinite[tid] = -1;
    if (tile_uneven(key0)) {
      lds_barrier();
      zero_infinite(key0, shared.values[0], &shared.infinite[0]);
    }
  }
  lds_barrier();
  if (second) lds_barrier();  // half a block behind the first group

  // Row of a transposing read, and the 16-byte part (its row's turn repeats every 4 rows).
  const int value_row = 4 * half + ((lane & 15) >> 2), value_column = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  floatx16 s[kHalves];
  bf16x8 p[2 * kHalves];
  int b0 = 0, b1 = 1, b2 = kBuffers - 1;  // buffers of this block, the next and the last
  float base = 0.0f, limit = __builtin_nanf(""), size = scale.size;
  for (int block = 0;; ++block) {
    const int key = key0 + block * kKeys;
    // Products: scores of this block, then the values of the last at its weights.
    // Parts of a row differ by an exclusive or of the lane's own: one instruction a
    // read, where addresses held in registers would cost the kernel its second wave.
    int key_at = key_part<D>(column, half), value_at = value_part<D>(value_row, value_column) + 8 * (lane & 1);
    asm volatile("" : "+v"(key_at), "+v"(value_at));
    const bool scores = block < blocks && wave_attends(key);
    const bool weighted = block > 0 && wave_attends(key - kKeys);
    constexpr int kProducts = kHalves * kSteps, kValueProducts = 2 * kHalves * kColumns;
    const uint8_t *k = shared.keys[b0], *v = shared.values[b2];
    const int after = kGroups == 2 ? b2 : b0;  // the buffer of the block after next
    auto key_fragment = [&](int n) {
      return *reinterpret_cast<const bf16x8*>(k + (key_at ^ (32 * (n % kSteps))) + 32 * (n / kSteps) * (2 * D));
    };
    auto value_fragment = [&](int n) {
      const uint8_t* at = v + (value_at ^ (64 * (n % kColumns))) + 16 * (n / kColumns) * (2 * D);
      const uint32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * (2 * D));
      return operand(lo[0], lo[1], hi[0], hi[1]);
    };
    if constexpr (kGroups == 2) __builtin_amdgcn_s_setprio(1);  // (the wave that multiplies goes first: 1 %)
    bf16x8 w[kAhead];
    if (scores) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) w[n] = key_fragment(n);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = 0.0f;
#pragma unroll
      for (int n = 0; n < kProducts; ++n) {
        s[n / kSteps] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[n % kAhead], qf[n % kSteps], s[n / kSteps], 0, 0, 0);
        if (n + kAhead < kProducts) w[n % kAhead] = key_fragment(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (weighted) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) w[n] = value_fragment(n);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kValueProducts; ++n) {
        const int e = n / kColumns, t = n % kColumns;
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[n % kAhead], p[e], o[t], 0, 0, 0);
        if (n + kAhead < kValueProducts) w[n % kAhead] = value_fragment(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (tile_uneven(key - kKeys) && shared.infinite[b2] == key - kKeys) add_infinite(key - kKeys);
    }
    if constexpr (kGroups == 2) __builtin_amdgcn_s_setprio(0);
    if (block >= blocks) break;
    // What was loaded beside the last weights: this block's values, the next one's keys.
    if (block > 0) {
      if constexpr (kE4m3)
        store_keys(shared.keys[b1]), store_values(shared.values[b0]);
      else
        wait_loads();
      if (tile_uneven(key)) zero_infinite(key, shared.values[b0], &shared.infinite[b0]);
    }
    lds_barrier();

    // Weights; loads of the keys after next and of the next values among them.
    const int page2 = page_of(key + 2 * kKeys, entry);
    entry = entry_of(key + 3 * kKeys);
    const uint64_t attended2 = __ballot(page2 >= 0);
    const uint8_t* key_rows = row_of(keys, a.k_page, a.k_token, key + 2 * kKeys, page2);
    const uint8_t* value_rows = row_of(values, a.v_page, a.v_token, key + kKeys, page1);
    const bool pieces = piecewise && attended2 == ~uint64_t{0} && attended1 == ~uint64_t{0};
    if (!pieces) {
      if (block + 2 < blocks) load_keys(key_rows, shared.keys[after]);
      if (block + 1 < blocks) load_values(value_rows, shared.values[b1]);
    }
    auto piece = [&](int n) {
      if constexpr (!kE4m3) {
        if (n < kLoads)
          load_piece(key_rows, k_lane, shared.keys[after], n);
        else
          load_piece(value_rows, v_lane, shared.values[b1], n - kLoads);
      }
    };
    auto weigh = [&](auto with_loads) {
      constexpr int kEvery = kHalves * 16 / (2 * kLoads);
      // (the packing of one copy is not the other's: made for both ahead of the branch, its results
      // were moved to the products' registers, 3 % of a chunk)
      if constexpr (decltype(with_loads)::value) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) asm volatile("" : "+v"(s[h]));
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (decltype(with_loads)::value)
            if ((16 * h + i) % kEvery == 0) piece((16 * h + i) / kEvery);
          sum += s[h][i];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          p[2 * h + e] = operand(pack_bf16x2(s[h][8 * e], s[h][8 * e + 1]), pack_bf16x2(s[h][8 * e + 2], s[h][8 * e + 3]),
                                 pack_bf16x2(s[h][8 * e + 4], s[h][8 * e + 5]), pack_bf16x2(s[h][8 * e + 6], s[h][8 * e + 7]));
      }
    };
    if (scores) {
      // Rows of the wave attend different keys of the block, or none of some: bit c
      // of the lane's mask is key c of the block.
      const bool uneven = wave_uneven(key) || attended != ~uint64_t{0};
      auto mask_of_row = [&] {
        const int newest = position - key, stale = oldest - key + 1;  // bits above and below them go
        uint64_t mask = kKeys == 32 ? attended & 0xffffffffu : attended;
        mask &= newest < 0 ? 0 : ~uint64_t{0} >> (newest < 63 ? 63 - newest : 0);
        mask &= stale <= 0 ? ~uint64_t{0} : (stale < 64 ? ~uint64_t{0} << stale : 0);
        return mask;
      };
      if (uneven) {
        const uint64_t mask = mask_of_row() >> (4 * half);
        const uint32_t mask_lo = static_cast<uint32_t>(mask), mask_hi = static_cast<uint32_t>(mask >> 32);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[h][i] = attended_or_nothing(s[h][i], h ? mask_hi : mask_lo, 8 * (i >> 2) + (i & 3));
      }
      float most = s[0][0];
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[h][i]);
      most = max_across_32(most) * scale.size;
      if (__any(!(most <= limit))) {
        const bool fresh = limit != limit;
        const bool attends = !uneven || mask_of_row() != 0;
        const bool raise = fresh ? attends : most > base;
        const float higher = raise ? fmaxf(most, kLowest) : base;
        const float shrink = raise && !fresh ? exp2_fast(base - higher) : 1.0f;
        base = higher;
        sum *= shrink;
#pragma unroll
        for (int t = 0; t < kColumns; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t][i] *= shrink;
        const bool coarse = __any(fabsf(base) >= kCoarse);
        if (!fresh || attends) limit = coarse ? -__builtin_huge_valf() : base + kSlack;
        size = coarse ? 1.0f : scale.size;
        if (coarse) {
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[h][i] *= scale.size;
        }
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = exp2_fast(fmaf(s[h][i], size, -base));
      if (pieces)
        weigh(std::true_type{});
      else
        weigh(std::false_type{});
    } else if (pieces) {
#pragma unroll
      for (int n = 0; n < 2 * kLoads; ++n) piece(n);
    }
    page1 = page2;
    attended = attended1, attended1 = attended2;
    const int last = b0;
    b0 = b1, b1 = kGroups == 2 ? b2 : last, b2 = last;
    lds_barrier();
  }
  if (kGroups == 2 && !second) lds_barrier();  // (as many as the second group)

  sum = sum_across_32(sum);
  const float top = limit != limit ? -__builtin_huge_valf() : base;  // (of a row that attends nothing)
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
  const bool nothing = top == -__builtin_huge_valf();
  const float inverse = value_scale / sum;
  uint16_t* out = a.out + static_cast<int64_t>(u.first_row + my_token) * a.out_row + my_head * a.out_head;
#pragma unroll
  for (int t = 0; t < kColumns; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      floatx4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = nothing ? 0.0f : o[t][4 * i + j] * inverse;
      store_row4(out + 32 * t + 8 * i + 4 * half, w);
    }
}

template <int D, bool kE4m3, int kGroups>
__global__ __launch_bounds__(4 * kGroups * kWave, D == 256 ? 1 : (D == 64 ? 3 : 2)) void paged_tile_kernel(PagedArgs a) {
  __shared__ union Shared {
    __device__ Shared() {}
    DecodeShared<D, 4 * kGroups> decode;
    TileShared<D, kGroups> tile;
  } shared;
  const int unit = static_cast<int>(blockIdx.x) / a.kv_heads, head = static_cast<int>(blockIdx.x) % a.kv_heads;
  if (unit < a.shares) {
    decode_share<D, kE4m3, 4 * kGroups>(a, unit, head, shared.decode);
  } else if (unit < a.shares + a.tile_units) {
    const PagedUnit u = paged_tile_unit<false>(a, unit - a.shares);
    if (u.live) tile_unit<D, kE4m3, kGroups>(a, u, head, shared.tile);
  } else {
    paged_zero_rest(a, static_cast<int>(blockIdx.x) - (a.tile_units + a.shares) * a.kv_heads, D);
  }
}

// A row's parts, added at the weights of their maxima: four columns of a thread.
struct Joined {
  float highest, total;
  floatx4 sum;
  __device__ void add(float top, float weights, const floatx4& part, float base) {
    const float weight = exp2_fast(top - base);
    total += weight * weights;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = fmaf(weight, part[k], sum[k]);
  }
  // Before parts of a maximum `higher`; what their weights are powers of two above.
  __device__ float raise(float higher) {
    const float base = higher == -__builtin_huge_valf() ? 0.0f : higher;
    const float shrink = highest == higher ? 1.0f : exp2_fast(highest - base);
    total *= shrink;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] *= shrink;
    highest = higher;
    return base;
  }
  __device__ void store(uint16_t* out, float value_scale) {
    const bool nothing = highest == -__builtin_huge_valf();
    const float inverse = value_scale / total;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = nothing ? 0.0f : sum[k] * inverse;
    store_row4(out, sum);
  }
};

// Every `stride`-th of the parts from `first` on, in the order of their keys, eight in
// flight.  Part n is at + n * step, but for the first of all: `lead` behind.
template <int D>
__device__ __forceinline__ Joined join_parts(const float* sums, const float2* stats, int64_t at, int64_t step, int64_t lead,
                                             int first, int stride, int parts, int d) {
  constexpr int kBatch = 8;
  Joined row = {-__builtin_huge_valf(), 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
  for (int s = first; s < parts; s += kBatch * stride) {
    float2 stat[kBatch];
    floatx4 w[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int n = min(s + b * stride, parts - 1);
      const int64_t from = at + n * step + (n == 0 ? lead : 0);
      stat[b] = stats[from];
      w[b] = *reinterpret_cast<const floatx4*>(sums + from * D + d);
    }
    float higher = row.highest;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) higher = s + b * stride < parts ? fmaxf(higher, stat[b].x) : higher;
    const float base = row.raise(higher);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (s + b * stride < parts) row.add(stat[b].x, stat[b].y, w[b], base);
  }
  return row;
}

// Workgroups 0 .. tiles * kv heads * (16-row parts): 16 rows of every `tiles`-th tile
// that is split.  Those behind them, of single tokens' tiles: `lanes` workgroups a
// tile, each 16 / lanes of its rows, a row's parts among `lanes` groups of threads
// (few tiles have many parts: a token's 60000 keys 78 us with one); or (lanes 0) one
// for each share that ends in a tile.
template <int D>
__global__ __launch_bounds__(4 * D) void paged_join_kernel(PagedArgs a, int tiles, int lanes, bool e4m3) {
  __shared__ Joined joined[4 * D];
  const int row_parts = a.tile_rows / 16;
  const int d = 4 * (static_cast<int>(threadIdx.x) % (D / 4)), r = static_cast<int>(threadIdx.x) / (D / 4);
  const int of_tiles = tiles * a.kv_heads * row_parts;
  const bool single = static_cast<int>(blockIdx.x) >= of_tiles;
  const int index = static_cast<int>(blockIdx.x) - (single ? of_tiles : 0);
  const int head = index % a.kv_heads;
  const float value_scale = e4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  auto out_of = [&](const PagedUnit& u, int token, int member) {
    return a.out + static_cast<int64_t>(u.first_row + token) * a.out_row + (head * a.group + member) * a.out_head + d;
  };
  if (single) {
    PagedShares shares;
    shares.start(a);
    PagedUnit u;
    int first, parts;  // workgroup of the tile's first part
    if (lanes > 0) {
      u = shares.find<true>(a, index / a.kv_heads / lanes);
      if (!u.live) return;
      first = u.from / shares.each, parts = (u.from + u.blocks - 1) / shares.each - first + 1;
    } else {
      // Of the shares that end in a tile, the one that does so first.
      first = index / a.kv_heads;
      const int64_t end = static_cast<int64_t>(first + 1) * shares.each;
      if (end >= shares.total) return;
      u = shares.find(a, static_cast<int>(end));
      if (!u.live || u.from == 0 || u.from > shares.each) return;
      parts = 1 + (u.blocks + shares.each - 1) / shares.each;
    }
    const int rows = lanes > 0 ? 16 / lanes : 16;
    if (parts == 1 || first < 0 || first > a.shares - parts) return;
    const int mine = r % rows + (lanes > 0 ? rows * (index / a.kv_heads % lanes) : 0), group = r / rows;
    const int member = 16 * (u.tile % a.slices) + mine;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * 16;
    Joined row = join_parts<D>(a.single_sums, a.single_stats, 2 * first * step + head * 16 + mine, 2 * step, step, group,
                               lanes > 0 ? lanes : 1, parts, d);
    if (lanes > 1) {
      joined[threadIdx.x] = row;
      __syncthreads();
      if (group > 0) return;
      for (int g = 1; g < lanes; ++g) {
        const Joined& other = joined[threadIdx.x + g * rows * (D / 4)];
        const float base = row.raise(fmaxf(row.highest, other.highest));
        row.add(other.highest, other.total, other.sum, base);
      }
    }
    if (member < a.group) row.store(out_of(u, u.tile / a.slices, member), value_scale);
    return;
  }
  const int row = 16 * (index / a.kv_heads % row_parts) + r;
  for (int t = index / (a.kv_heads * row_parts);; t += tiles) {
    const PagedUnit u = paged_tile_unit<true>(a, t);
    if (!u.live) return;
    const int m = u.tile * a.tile_rows + row;
    if (m >= u.tokens * a.group) continue;
    const int token = m / a.group;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.tile_rows;
    join_parts<D>(a.tile_sums, a.tile_stats, u.part * step + head * a.tile_rows + row, step, 0, 0, 1, u.splits, d)
        .store(out_of(u, token, m - token * a.group), value_scale);
  }
}

// How a call is cut, as far as the host knows its sizes.  Measured (us):
//   kAlone: a token's 333 keys by one workgroup a kv head 7.8, cut in three and joined 10.4;
//   workgroups a CU for single tokens: 52 x 2048 keys of 256 columns 39.0 with one, 40.2
//   with two, 47.5 with three; 16 x 32768 e4m3 keys 193, 140, 141 (four: 155); a mixed
//   step, whose tiles take the other place, 37.9 with one, 38.3 with two (over 2048 keys;
//   with long contexts one is too few: those 16 with a prompt of 16 rows 164, alone 134);
//   kLeastShare: those 52 tokens 40.2 with two blocks or four, 48 with eight;
//   kTwoGroupRows: a prompt of 8192 (32768 packed rows) 300 with tiles of two groups, 334
//   with one; eight of 1000 (4000) 102 and 104; sixteen of 512 (2048) 85 and 80 (all
//   three are faster since, alike).
constexpr int kCus = 256;
constexpr int kAlone = 512;          // keys that are not worth a second launch
constexpr int kLeastShare = 4;       // fewest blocks of a share
constexpr int kTwoGroupRows = 4096;  // packed rows of the longest sequence

struct PagedPlan {
  bool all_single, split_tiles, split_shares;
  int slices, tile_rows, tile_tokens, share_shift, shares, least, target, work_shift;
  int64_t single_tiles, tiles, tile_units, single_parts, tile_parts;
};

PagedPlan paged_plan(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences, int32_t max_length) {
  PagedPlan p = {};
  const int64_t group = q_heads / c->kv_heads;
  const int64_t capacity = static_cast<int64_t>(c->max_pages) * c->page_size;
  const int64_t some = sequences < rows ? sequences : rows;
  p.all_single = max_length <= 1;
  p.slices = static_cast<int>((group + 15) / 16);
  // Tiles of two groups where they alone fill the card; a launch holds 2^32 threads, of which
  // 512 for a sequence's and a kv head's last tile.
  const bool two_groups = c->head_dim == 128 && rows * q_heads >= int64_t{kCus} * 2 * kGroupRows &&
                          max_length * group >= kTwoGroupRows && some * c->kv_heads <= (int64_t{1} << 22);
  p.tile_rows = two_groups ? 2 * kGroupRows : kGroupRows;
  p.tile_tokens = p.all_single ? 1 : static_cast<int>(p.tile_rows / group + 2);
  // Single tokens: blocks of 64 keys; one block a tile where no slot holds more keys
  // than are worth a second launch; larger where all of them could be 2^30 and more.
  const int64_t single_tiles = p.single_tiles = (p.all_single ? rows : some) * p.slices;
  p.share_shift = 6;
  while (capacity <= kAlone && capacity > 1 << p.share_shift) ++p.share_shift;
  while ((((capacity - 1) >> p.share_shift) + 1) * single_tiles >= int64_t{1} << 30) ++p.share_shift;
  const int64_t blocks = ((capacity - 1) >> p.share_shift) + 1;
  const int resident = (!p.all_single ? 1 : (c->head_dim == 64 ? 4 : 2)) * kCus / c->kv_heads;
  p.least = blocks > 1 ? kLeastShare : 1;
  // No more workgroups than the blocks can give work to.
  const int64_t useful = (single_tiles * blocks + p.least - 1) / p.least;
  p.shares = sequences == 0 ? 0 : static_cast<int>(useful < resident ? useful : (resident > 0 ? resident : 1));
  p.split_shares = p.shares > 1 && blocks > 1;
  p.single_parts = p.split_shares ? 2 * static_cast<int64_t>(p.shares) : 0;
  // Tiles of more rows.
  p.target = (two_groups ? 1 : 2) * kCus / c->kv_heads;
  if (p.target < 1) p.target = 1;
  if (!p.all_single && sequences > 0) {
    p.tiles = rows * group / p.tile_rows + some;
    p.split_tiles = (capacity + kKeyBlock - 1) / kKeyBlock > kLeastSplit;
    p.tile_units = p.tiles + (p.split_tiles ? p.target : 0);
    const int64_t most = (capacity + kKeyBlock - 1) / kKeyBlock;
    while (p.tiles * (((most - 1) >> p.work_shift) + 1) >= (int64_t{1} << 31)) ++p.work_shift;
    p.tile_parts = p.split_tiles ? 2 * static_cast<int64_t>(p.target) : 0;
  }
  return p;
}

int64_t workspace_rows(const PagedPlan& p, const d3_paged_cache* c) {
  return (p.single_parts * 16 + p.tile_parts * p.tile_rows) * c->kv_heads;
}

bool attention_suited(const d3_paged_cache* c, int64_t rows, int32_t q_heads, int32_t sequences) {
  // (so many heads that 256 threads of a tile and 1024 of a join's sixteen rows stay below 2^32)
  return (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && rows * q_heads <= (int64_t{1} << 23) &&
         sequences <= 65536 && c->kv_heads <= 65536;
}

void launch_paged_tiles(const PagedArgs& a, int head_dim, bool e4m3, bool zero_rest, hipStream_t stream) {
  const unsigned workgroups = paged_workgroups(a, zero_rest);
  auto run = [&](auto kernel, int groups) {
    hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(4 * groups * kWave), 0, stream, a);
  };
  if (head_dim == 64)
    e4m3 ? run(paged_tile_kernel<64, true, 1>, 1) : run(paged_tile_kernel<64, false, 1>, 1);
  else if (head_dim == 256)
    e4m3 ? run(paged_tile_kernel<256, true, 1>, 1) : run(paged_tile_kernel<256, false, 1>, 1);
  else if (a.tile_rows == kGroupRows)
    e4m3 ? run(paged_tile_kernel<128, true, 1>, 1) : run(paged_tile_kernel<128, false, 1>, 1);
  else
    e4m3 ? run(paged_tile_kernel<128, true, 2>, 2) : run(paged_tile_kernel<128, false, 2>, 2);
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
  D3_REQUIRE(__builtin_isfinite(scale * kLog2E), "paged_attention: scale times log2(e) must be finite");
  D3_REQUIRE((sequence_slots_dtype == D3_DTYPE_I32 || sequence_slots_dtype == D3_DTYPE_I64) &&
                 (lengths_dtype == D3_DTYPE_I32 || lengths_dtype == D3_DTYPE_I64),
             "paged_attention: slots and lengths must be int32 or int64");
  D3_SUPPORTED(attention_suited(cache, rows, q_heads, sequences),
               "paged_attention: head dim %d (64, 128 or 256), %lld rows of %d heads, %d kv heads, %d sequences", cache->head_dim,
               static_cast<long long>(rows), q_heads, cache->kv_heads, sequences);
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
  a.k_page = static_cast<uint32_t>(cache->key_page_stride * size), a.k_token = static_cast<uint32_t>(cache->key_token_stride * size);
  a.k_head = cache->key_head_stride * size;
  a.v_page = static_cast<uint32_t>(cache->value_page_stride * size), a.v_token = static_cast<uint32_t>(cache->value_token_stride * size);
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
  a.slices = p.slices, a.all_single = p.all_single, a.tile_rows = p.tile_rows, a.tile_tokens = p.tile_tokens;
  a.scale = scale * kLog2E;
  a.window = static_cast<int>(window < 0 ? 0 : (window < 0x7fffffff ? window : 0x7fffffff));
  a.share_shift = p.share_shift, a.shares = p.shares, a.least = p.least;
  a.target = p.target, a.work_shift = p.work_shift, a.splitting = p.split_tiles;
  a.target_inverse = p.target > 1 ? static_cast<uint32_t>((uint64_t{1} << 32) / p.target + 1) : 0xffffffffu;
  a.tile_units = static_cast<int>(p.tile_units);
  a.tile_parts = static_cast<int>(p.tile_parts);
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
    const int few = p.target < 8 ? 1 : p.target / 8;  // (of the tiles, up to p.target are split)
    const int tiles = p.split_tiles ? static_cast<int>(p.tiles < few ? p.tiles : few) : 0;
    // Single tokens' tiles: by their number where they are fewer than the shares.
    int lanes = 0;
    int64_t singles = p.split_shares ? p.shares - 1 : 0;
    if (p.split_shares && p.single_tiles <= p.shares) {
      lanes = 1;
      while (lanes < 16 && p.single_tiles * lanes * 8 < p.shares) lanes *= 2;  // (a thread's parts in one batch)
      singles = p.single_tiles * lanes;
    }
    const dim3 grid(static_cast<unsigned>((tiles * (p.tile_rows / 16) + singles) * cache->kv_heads)), block(4 * cache->head_dim);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), a, tiles, lanes, e4m3); };
    if (cache->head_dim == 64)
      run(paged_join_kernel<64>);
    else if (cache->head_dim == 128)
      run(paged_join_kernel<128>);
    else
      run(paged_join_kernel<256>);
  }
  D3_LAUNCHED("paged_attention");
}
