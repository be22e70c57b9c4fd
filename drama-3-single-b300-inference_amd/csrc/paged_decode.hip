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
// Bound by HBM: every key and value is read once.  The four waves of a workgroup
// take blocks of 32 keys in turn, each with its own running softmax and no
// barrier until the end, where their rows are added in LDS; the next block's
// keys and values are in flight while one is multiplied.
#include "paged_attention.h"

namespace d3 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = 32;  // of a wave's step

template <int D, bool kE4m3>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void paged_decode_kernel(PagedArgs a) {
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowParts = D * kBytes / 16;      // 16-byte parts of a cached row
  constexpr int kKeyLoads = 2 * (kRowParts / 4);  // a lane's: key lane % 16 of two tiles, every fourth part
  constexpr int kKeysALoad = kWave / kRowParts;   // value rows a load covers
  constexpr int kValueLoads = kKeys / kKeysALoad;
  constexpr int kSteps = D / 32, kTiles = D / 16;
  constexpr int kSwizzle = D >= 128 ? 7 : 3;
  constexpr int kShift = D >= 128 ? 0 : 1;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves][kKeys * D * 2];
  __shared__ float2 wave_stats[kWaves][16];

  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int column = lane & 15, g = lane >> 4;
  const int head = static_cast<int>(blockIdx.x) % a.kv_heads;
  if (a.zero_rest) paged_zero_rest(a, blockIdx.x, gridDim.x, D);
  const PagedUnit u = paged_unit<false>(a, static_cast<int>(blockIdx.x) / a.kv_heads);
  if (!u.live) return;
  const int token = u.tile / a.slices, slice = u.tile % a.slices;
  const int heads = min(16, a.group - 16 * slice);  // live columns
  const int row = u.first_row + token;
  const int q_head0 = head * a.group + 16 * slice;

  // Q^T operand: column = head, elements by the keys' order of the contraction.
  // bf16 keys: step s, element j of group g is column 32 s + 8 g + j; e4m3 ones
  // come 16 at a time: 64 (s / 2) + 16 g + 8 (s % 2) + j.
  bf16x8 qf[kSteps];
  {
    const uint16_t* q = a.q + row * a.q_row + (q_head0 + min(column, heads - 1)) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = kE4m3 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const RowVector4*>(q + d));
    }
  }
  const int64_t slot = paged_index(a.sequence_slots, a.slots_64, u.sequence);
  PagedKeys range = paged_keys(a, u, token, token);
  if (slot < 0 || slot >= a.slots) range.high = range.low;
  const int32_t* pages = a.page_table + (slot < 0 || slot >= a.slots ? 0 : slot) * a.table_stride;
  const float key_scale = a.scale * (kE4m3 && a.k_scales != nullptr ? a.k_scales[head] : 1.0f);
  const uint8_t* keys = a.keys + head * a.k_head;
  const uint8_t* values = a.values + head * a.v_head;
  const int in_page = (1 << a.page_shift) - 1;

  floatx4 o[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) o[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  float top = -__builtin_huge_valf(), sum = 0.0f;

  // Blocks from the aligned one that holds the first key; wave w takes every fourth.
  const int first = range.low & ~(kKeys - 1);
  auto page_of = [&](int key) -> int {  // of lane's key % 32, -1 where nothing is attended
    const int at = key + (lane & (kKeys - 1));
    const bool in = at >= range.low && at < range.high;
    const int page = pages[in ? at >> a.page_shift : 0];
    return in && static_cast<uint32_t>(page) < a.pages ? page : -1;
  };
  int32x4 kr[kKeyLoads], vr[kValueLoads];
  auto load_keys = [&](int key, int page) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int mine = 16 * t + column;
      const int p = __shfl(page, mine, kWave);
      const uint8_t* at = keys + p * a.k_page + ((key + mine) & in_page) * a.k_token + 16 * g;
      if (p < 0) at = paged_nothing;
#pragma unroll
      for (int i = 0; i < kRowParts / 4; ++i)
        kr[t * (kRowParts / 4) + i] = *reinterpret_cast<const int32x4*>(at + 64 * i);
    }
  };
  auto load_rows = [&](int key, int page) {
#pragma unroll
    for (int i = 0; i < kValueLoads; ++i) {
      const int mine = kKeysALoad * i + lane / kRowParts;
      const int p = __shfl(page, mine, kWave);
      const uint8_t* at = values + p * a.v_page + ((key + mine) & in_page) * a.v_token + 16 * (lane % kRowParts);
      if (p < 0) at = paged_nothing;
      vr[i] = *reinterpret_cast<const int32x4*>(at);
    }
  };

  int key = first + wave * kKeys;
  int page = page_of(key);
  if (key < range.high) {
    load_keys(key, page);
    load_rows(key, page);
  }
  int next_page = page_of(key + kWaves * kKeys);
  uint8_t* mine = lds[wave];
  for (; key < range.high; key += kWaves * kKeys) {
    const uint32_t attended = static_cast<uint32_t>(__ballot(page >= 0));
    // S^T of two 16-key tiles
    floatx4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
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
    if (next < range.high) load_keys(next, next_page);
    // The running softmax, in powers of two
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] *= key_scale;
    if (attended != 0xffffffffu) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[t][i] = (attended >> (16 * t + 4 * g + i)) & 1u ? s[t][i] : -__builtin_huge_valf();
    }
    float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    most = max_across_16(most);
    if (__any(most > top)) {
      const float higher = fmaxf(top, most);
      const float shrink = top == higher ? 1.0f : exp2_fast(top - higher);
      top = higher;
      sum *= shrink;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] *= shrink;
    }
    const float base = top == -__builtin_huge_valf() ? 0.0f : top;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = exp2_fast(s[t][i] - base);
        sum += s[t][i];
      }
    const bf16x8 p = operand(pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]),
                             pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3]));
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
    next_page = page_of(next + kWaves * kKeys);
    // O^T += V^T P^T
    const int r = 4 * g + (column >> 2);
    const int turn = 2 * ((r >> kShift) & kSwizzle);  // row r + 16 has the same
    const uint8_t* at = mine + r * (2 * D) + 8 * (column & 1);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int part = ((2 * t + ((column >> 1) & 1)) ^ turn) << 4;
      const uint32x2 lo = read_transposed(at + part), hi = read_transposed(at + part + 16 * 2 * D);
      o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(lo[0], lo[1], hi[0], hi[1]), p, o[t], 0, 0, 0);
    }
  }

  // The waves' rows to LDS (fp32 [column][D], a wave's values' space), then one
  // pass adds them at the weights of their maxima.
  sum = sum_across_16(sum);
  if (g == 0) wave_stats[wave][column] = make_float2(top, sum);
  float* sums = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
    *reinterpret_cast<floatx4*>(sums + column * D + ((16 * t + 4 * g) ^ (4 * (column & 7)))) = o[t];
  __syncthreads();
  constexpr int kParts = D / 4;
  const float value_scale = kE4m3 && a.v_scales != nullptr ? a.v_scales[head] : 1.0f;
  for (int i = static_cast<int>(threadIdx.x); i < heads * kParts; i += kThreads) {
    const int c = i / kParts, d = 4 * (i % kParts);
    float highest = -__builtin_huge_valf();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, wave_stats[w][c].x);
    const float base = highest == -__builtin_huge_valf() ? 0.0f : highest;
    float total = 0.0f;
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 stat = wave_stats[w][c];
      const float weight = exp2_fast(stat.x - base);
      total += weight * stat.y;
      const floatx4 part = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(lds[w]) + c * D + (d ^ (4 * (c & 7))));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmaf(weight, part[k], v[k]);
    }
    if (u.splits > 1) {
      const int64_t at = (static_cast<int64_t>(u.partial + u.split) * a.kv_heads + head) * 16 + c;
      *reinterpret_cast<floatx4*>(a.sums + at * D + d) = v;
      if (d == 0) a.stats[at] = make_float2(highest, total);
    } else {
      const float inverse = total == 0.0f ? 0.0f : value_scale / total;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : v[k] * inverse;
      store_row4(a.out + row * a.out_row + (q_head0 + c) * a.out_head + d, v);
    }
  }
}

}  // namespace

void launch_paged_decode(const PagedArgs& a, int head_dim, bool e4m3, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.max_units) * a.kv_heads), block(kThreads);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  if (head_dim == 64)
    e4m3 ? run(paged_decode_kernel<64, true>) : run(paged_decode_kernel<64, false>);
  else if (head_dim == 128)
    e4m3 ? run(paged_decode_kernel<128, true>) : run(paged_decode_kernel<128, false>);
  else
    e4m3 ? run(paged_decode_kernel<256, true>) : run(paged_decode_kernel<256, false>);
}

}  // namespace d3
