// Products of MXFP4 rows with packed MXFP4 weights: dense, grouped by expert
// over ragged boundaries, and the two products of the routed SwiGLU experts.
//
// out[r, j] = sum_k a[r, k] w[j, k] on mfma_scale_f32_16x16x128_f8f6f4 with
// both operands e2m1: a lane's operand is exactly one block of 32 elements,
// so its e8m0 scale is the instruction's own scale operand and no rescaling
// is left to the vector unit.  The products are exact and the sums fp32 (6e-8
// of sum |products| measured over scales that differ by 2^40).  Weights are
// the first operand: an output lane holds one row of a and four consecutive
// weight rows of each 16-row tile, as the packed row orders place them.
#include <type_traits>
#include <utility>

#include "mxfp4.h"
#include "status.h"

namespace d3 {
namespace {

constexpr int kMxWaves = 4;
constexpr int kMxThreads = kMxWaves * kWave;

enum MxEpilogue {
  kMxBf16,  // bf16 rows at the item's rows
  kMxAct,   // silu(gate) * up quantised to MXFP4 rows at the item's rows (gate-up order)
  kMxF32,   // fp32 rows at sorted[row]
};

struct MxGemm {
  const uint8_t* w;  // packed codes [E][row groups][steps][8 KiB]
  const uint8_t* ws;
  int n;
  int row_groups;
  int steps;
  const uint8_t* a;  // quantised rows (operand layout, `steps` steps)
  int64_t a_rows;
  const uint8_t* as;
  const uint16_t* x;  // or the rows themselves, bf16 [rows][k], quantised by the wave that multiplies them
  int64_t x_stride;
  int k_blocks;       // k / 32
  const int4* items;  // {expert (-1: zero rows), first row, rows, -}; nullptr: one expert, `rows` in order
  const int32_t* num_items;
  int max_items;
  int rows;
  const int32_t* sorted;  // route list: row of a = sorted[row] / top_k (kMxAct), row of out = sorted[row] (kMxF32);
  int top_k;              // nullptr: the identity
  const void* ids;        // kMxPairs, kMxScan: expert of each (row, rank) pair (kMxScan: of `rows` pairs)
  int ids_i64;
  int experts;
  const int32_t* bounds;  // kMxGroups: the groups' boundaries
  int zero_rest;
  void* out;
  int64_t out_stride;  // elements (kMxAct: the row's width)
  bool out_past;  // kMxBf16, tiled: more than the L2s hold, stored past them
  uint8_t* out_scales;  // kMxAct: out and out_scales in the operand layout
};

// One MFMA with the scales in byte SA of `sa` and byte SB of `sb`.
template <int SA, int SB>
__device__ __forceinline__ floatx4 mfma_fp4(const int32x4& a, const int32x4& b, const floatx4& c, uint32_t sa, uint32_t sb) {
  const int32x8 av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  const int32x8 bv = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, kMxLow, kMxLow, SA, static_cast<int>(sa), SB,
                                                          static_cast<int>(sb));
}

template <int SB>
__device__ __forceinline__ void mfma_tiles(const int32x4 (&a)[4], const int32x4& b, floatx4 (&c)[4], uint32_t sa, uint32_t sb) {
  c[0] = mfma_fp4<0, SB>(a[0], b, c[0], sa, sb);
  c[1] = mfma_fp4<1, SB>(a[1], b, c[1], sa, sb);
  c[2] = mfma_fp4<2, SB>(a[2], b, c[2], sa, sb);
  c[3] = mfma_fp4<3, SB>(a[3], b, c[3], sa, sb);
}

__device__ __forceinline__ int4 mx_item(const MxGemm& g, int index, int item_rows) {
  if (g.items == nullptr) {
    const int start = index * item_rows;
    return make_int4(0, start, min(item_rows, g.rows - start), 0);
  }
  // Read with the count, not after it: every index below max_items is in the list.
  const int live = *g.num_items;
  const int4 item = g.items[min(index, g.max_items - 1)];
  return index < live ? item : make_int4(0, 0, 0, 0);
}

__device__ __forceinline__ MxWords4 mx_pack8(const float* v) {
  MxWords4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w.w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  return w;
}

// Eight 16-bit values at columns f .. of a row of n.
__device__ __forceinline__ void mx_store16(uint16_t* out, int f, int n, const MxWords4& v, bool past = false) {
  if (f + 8 <= n) {
    if (past)  // uniform
      __builtin_nontemporal_store(__builtin_bit_cast(MxVector4, v), reinterpret_cast<MxVector4*>(out + f));
    else
      *reinterpret_cast<MxWords4*>(out + f) = v;
    return;
  }
  uint64_t lo = v.w[0] | (static_cast<uint64_t>(v.w[1]) << 32), hi = v.w[2] | (static_cast<uint64_t>(v.w[3]) << 32);
#pragma unroll 1
  for (int i = f; i < n; ++i) {
    out[i] = static_cast<uint16_t>(lo);
    lo = (lo >> 16) | (hi << 48);
    hi >>= 16;
  }
}

// The four tiles of one row of `a` (this lane's row `row` of the item's list, or
// the row itself without one, live or not) for row group rg.
template <int kEpi>
__device__ __forceinline__ void mx_store(const MxGemm& g, const floatx4 (&c)[4], int rg, int row, bool live, int group) {
  if constexpr (kEpi == kMxBf16 || kEpi == kMxF32) {
    if (!live) return;
    int64_t to = row;
    if (kEpi == kMxF32 && g.sorted != nullptr) to = g.sorted[row];  // uniform
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int f = kMxRows * rg + 32 * p + 8 * group;
      if constexpr (kEpi == kMxF32) {  // whole row groups: n is a multiple of 128
        floatx4* out = reinterpret_cast<floatx4*>(static_cast<float*>(g.out) + to * g.out_stride + f);
        out[0] = c[2 * p];
        out[1] = c[2 * p + 1];
      } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c[2 * p + i / 4][i % 4];
        mx_store16(static_cast<uint16_t*>(g.out) + to * g.out_stride, f, g.n, mx_pack8(v));
      }
    }
  } else if constexpr (kEpi == kMxAct) {
    // Gate (tiles 0, 1) and up (tiles 2, 3) of columns 32 rg + 8 group + i;
    // the four groups of a row hold one block of 32.  Nothing is rounded
    // between the products and the codes.
    float gate[8], up[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gate[i] = c[i / 4][i % 4];
      up[i] = c[2 + i / 4][i % 4];
    }
    swiglu_values<8>(gate, up, v);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = MaxU32::apply(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    amax = MaxU32::apply(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16)));
    amax = MaxU32::apply(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32)));
    const uint32_t code = mx_scale_code(amax);
    const uint32_t word = mx_codes8(v, mx_inverse(code));
    if (!live) return;
    const uint32_t blocks = static_cast<uint32_t>(g.out_stride) / kMxBlock;
    const int64_t first = static_cast<int64_t>(row) * ((blocks + 7) / 8);  // in steps
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.out) + first * kMxOperandCodes + rg * (kMxBlock / 2) + 4 * group) = word;
    if (group == 0) mx_operand_scale(g.out_scales + first * kMxOperandScales, rg, blocks, code);
  }
}

// Columns first .. first + count (a multiple of 8) of an item's rows as zeros,
// eight a thread: 199 rows of no group beside 4 of 60 groups, N 1040, took 21.6
// us by single columns and a row at a time, 9.7 so (4.7 the kernel).
__device__ __forceinline__ void mx_zero_rows(const MxGemm& g, const int4& item, int first, int count) {
  const int units = min(count, g.n - first + 7) / 8;
  const MxWords4 zero = {};
  for (int64_t u = threadIdx.x; u < static_cast<int64_t>(item.z) * units; u += kMxThreads) {
    const int64_t r = u / units;
    uint16_t* out = static_cast<uint16_t*>(g.out) + (item.y + r) * g.out_stride;
    mx_store16(out, first + 8 * static_cast<int>(u - r * units), g.n, zero, false);
  }
}

// One lane's operand (one block of 32) of a bf16 row: no other lane's values
// are needed for its scale.
struct MxOperand {
  int32x4 codes;
  uint32_t scale;
};
__device__ __forceinline__ MxOperand mx_operand_bf16(const uint16_t* x) {
  MxWords4 raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = reinterpret_cast<const MxWords4*>(x)[i];
  const uint16x2 amax = mx_amax_bf16<16>(&raw[0].w[0]);
  MxOperand op;
  op.scale = mx_scale_code(MaxU32::apply(amax[0], amax[1]) << 16);
  const float scale = mx_scale(op.scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) op.codes[i] = static_cast<int>(mx_codes8_bf16(raw[i].w, scale));
  return op;
}

__device__ __forceinline__ int64_t mx_pair_expert(const MxGemm& g, int64_t pair) {
  return g.ids_i64 ? static_cast<const int64_t*>(g.ids)[pair] : static_cast<const int32_t*>(g.ids)[pair];
}

// Few rows an item (up to 16 kRT): the weights stream from memory once, each
// wave a share of the contraction.  A workgroup's four waves are kMxWaves /
// kSplit row groups by kSplit interleaved slices of the steps; the slices'
// fp32 sums meet in LDS (`part`) and are added in slice order.
// kDirect: the rows are bf16 and every wave quantises the operands it
// multiplies: about 50 vector instructions an operand against a launch of
// its own, which pays up to two row tiles.
// kOnce: weights that one item reads are loaded non-temporally (moe 64 rows E256
// 78.8 -> 72.0 us, grouped 384 rows E128 38.9 -> 37.4).
// kListed: the item's rows are those that `list` names (pairs), and so are the
// rows of what it stores.
template <int kRT, int kEpi, int kSplit, bool kDirect, bool kOnce, bool kListed = false>
__device__ __forceinline__ void mx_stream_item(const MxGemm& g, const int4& item, int block, floatx4* part,
                                               const int32_t* list = nullptr) {
  constexpr int kGroups = kMxWaves / kSplit;
  const int lane = lane_id(), row16 = lane & 15, group = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int slice = wave % kSplit;
  const int rg = block * kGroups + wave / kSplit;
  const int rg_read = min(rg, g.row_groups - 1);
  const int count = min(item.z, 16 * kRT);

  // Rows past the item read its last row; their sums are dropped.
  const uint8_t* codes[kRT];
  const uint8_t* scales[kRT];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    int64_t row = item.y + min(16 * rt + row16, count - 1);
    if constexpr (kListed) row = list[row];
    if constexpr (kEpi == kMxAct) row = (g.sorted ? g.sorted[row] : static_cast<int>(row)) / g.top_k;
    if constexpr (kDirect) {
      codes[rt] = reinterpret_cast<const uint8_t*>(g.x + row * g.x_stride);
    } else {
      codes[rt] = g.a + row * g.steps * kMxOperandCodes + 16 * group;
      scales[rt] = g.as + row * g.steps * kMxOperandScales + 4 * (group & 1);
    }
  }
  const int64_t base = static_cast<int64_t>(item.x) * g.row_groups + rg_read;
  const int32x4* w = reinterpret_cast<const int32x4*>(g.w + base * g.steps * kMxStepCodes) + lane;
  const uint2* ws = reinterpret_cast<const uint2*>(g.ws + base * g.steps * kMxStepScales) + lane;

  auto store_row = [&](int rt) {
    const int at = item.y + 16 * rt + row16;
    return kListed ? list[min(at, item.y + count - 1)] : at;
  };

  floatx4 acc[kRT][4];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[rt][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int step = slice; step < g.steps; step += kSplit) {
    int32x4 wf[2][4];
    const int32x4* wp = w + static_cast<int64_t>(step) * (kMxStepCodes / 16);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        wf[h][t] = kOnce ? __builtin_nontemporal_load(wp + (4 * h + t) * kWave) : wp[(4 * h + t) * kWave];
    const uint2 wsc = ws[static_cast<int64_t>(step) * (kMxStepScales / 8)];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      if constexpr (kDirect) {
        // The padded half of the last step reads the first half again, at
        // scale 2^-127 (the weights are zeros there).
        const bool more = 8 * step + 4 < g.k_blocks;  // uniform
        const uint16_t* x = reinterpret_cast<const uint16_t*>(codes[rt]) + kMxStep * step + kMxBlock * group;
        const MxOperand lo = mx_operand_bf16(x);
        MxOperand hi = mx_operand_bf16(more ? x + 4 * kMxBlock : x);
        mfma_tiles<0>(wf[0], lo.codes, acc[rt], wsc.x, lo.scale);
        mfma_tiles<0>(wf[1], hi.codes, acc[rt], wsc.y, more ? hi.scale : 0u);
      } else {
        const uint32_t sb =
            *reinterpret_cast<const uint32_t*>(scales[rt] + kMxOperandScales * step) >> (8 * (group >> 1));
        const int32x4* b = reinterpret_cast<const int32x4*>(codes[rt] + kMxOperandCodes * step);
        mfma_tiles<0>(wf[0], b[0], acc[rt], wsc.x, sb);
        mfma_tiles<2>(wf[1], b[4], acc[rt], wsc.y, sb);
      }
    }
  }

  if constexpr (kSplit > 1) {
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
      for (int t = 0; t < 4; ++t) part[((wave * kRT + rt) * 4 + t) * kWave + lane] = acc[rt][t];
    __syncthreads();
    const int first = wave - slice;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      if (rt % kSplit != slice) continue;
      floatx4 sum[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        sum[t] = part[((first * kRT + rt) * 4 + t) * kWave + lane];
#pragma unroll
        for (int s = 1; s < kSplit; ++s) sum[t] += part[(((first + s) * kRT + rt) * 4 + t) * kWave + lane];
      }
      if (rg < g.row_groups)
        mx_store<kEpi>(g, sum, rg, store_row(rt), 16 * rt + row16 < count, group);
    }
  } else {
    if (rg >= g.row_groups) return;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
      mx_store<kEpi>(g, acc[rt], rg, store_row(rt), 16 * rt + row16 < count, group);
  }
}

// Where a streaming workgroup's rows come from.
enum MxSource {
  kMxList,   // the work items (or the rows in order)
  kMxPairs,  // an item per (row, rank) pair: few pairs, no route sort
  kMxScan,   // the pairs of an expert, found among all of them by its workgroups: no route sort either
  kMxGroups, // the groups of the boundaries, one or two row tiles at a time
};

// Routes without a sort: the workgroups of an expert find its pairs among all of
// them, and multiply the first 16.  An expert with more has a workgroup of its
// own for each further 16; there are as many of those as pairs can fill, at the
// front of the grid, and each finds its place from the experts' counts.
constexpr int kMxScanPairs = 5 * kMxThreads;
constexpr int kMxScanRounds = kMxScanPairs / kMxThreads;
constexpr int kMxMaxExperts = 512;
struct MxScan {
  int32_t list[kMxScanPairs];
  int counts[kMxMaxExperts];
  int tally[kMxScanRounds][kMxWaves];
  int expert, tile;
};
// An expert of c pairs has (c - 1) / 16 further tiles.
__host__ __device__ constexpr int mx_scan_extra(int pairs) { return pairs / 16; }

// The pairs of `expert` in ascending order; returns how many.
__device__ __forceinline__ int mx_scan_pairs(const MxGemm& g, int expert, MxScan& scan) {
  const int wave = threadIdx.x / kWave, rounds = (g.rows + kMxThreads - 1) / kMxThreads;
  int64_t id[kMxScanRounds];
  uint64_t hit[kMxScanRounds];
#pragma unroll
  for (int j = 0; j < kMxScanRounds; ++j)
    if (j < rounds) id[j] = mx_pair_expert(g, min(j * kMxThreads + static_cast<int>(threadIdx.x), g.rows - 1));
#pragma unroll
  for (int j = 0; j < kMxScanRounds; ++j)
    if (j < rounds) {
      hit[j] = __ballot(id[j] == expert && j * kMxThreads + static_cast<int>(threadIdx.x) < g.rows);
      if (lane_id() == 0) scan.tally[j][wave] = __builtin_popcountll(hit[j]);
    }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int j = 0; j < kMxScanRounds; ++j)
    if (j < rounds) {
      int before = total;
#pragma unroll
      for (int w = 0; w < kMxWaves; ++w) {
        const int n = scan.tally[j][w];
        before += w < wave ? n : 0;
        total += n;
      }
      if (hit[j] >> lane_id() & 1)
        scan.list[before + __builtin_popcountll(hit[j] & ((uint64_t{1} << lane_id()) - 1))] =
            j * kMxThreads + static_cast<int>(threadIdx.x);
    }
  __syncthreads();
  return total;
}

// Expert and tile (1, ..) of the further tile `index`, into `scan`; expert -1: there is none.
__device__ __forceinline__ void mx_scan_further(const MxGemm& g, int index, MxScan& scan) {
  static_assert(kMxMaxExperts == 2 * kMxThreads, "two experts a thread");
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  scan.counts[2 * tid] = scan.counts[2 * tid + 1] = 0;
  if (tid == 0) scan.expert = -1;
  __syncthreads();
  for (int at = tid; at < g.rows; at += kMxThreads) {
    const int64_t id = mx_pair_expert(g, at);
    if (id >= 0 && id < g.experts) atomicAdd(&scan.counts[id], 1);
  }
  __syncthreads();
  auto further = [&](int e) { return max((scan.counts[e] + 15) / 16 - 1, 0); };
  const int n0 = further(2 * tid), n1 = further(2 * tid + 1);
  int sum = n0 + n1;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int v = __shfl_up(sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == kWave - 1) scan.tally[0][wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += scan.tally[0][w];
  const int first = sum - n0 - n1;
  if (index >= first && index < first + n0)
    scan.expert = 2 * tid, scan.tile = 1 + index - first;
  else if (index >= first + n0 && index < sum)
    scan.expert = 2 * tid + 1, scan.tile = 1 + index - first - n0;
  __syncthreads();
}

// Two row tiles are held to four waves a SIMD (384 rows over 128 groups 37.7 ->
// 34.8 us; to five, with spills, 45); one tile has them anyhow, and asked for more
// loses in skewed batches what it gains in even ones.
template <int kRT, int kEpi, int kSplit, bool kDirect, int kSource>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(kRT > 1 ? 4 : 1))) void mx_stream_kernel(MxGemm g, int blocks) {
  constexpr int kGroups = kMxWaves / kSplit;
  // One matrix is read by every item; an expert's mostly by one (but a call of
  // few pairs or workgroups is short of latency, not of cache: non-temporal
  // loads cost one token's gate and up product 5.5 -> 7.2 us where its experts
  // are cached, and kMxScan's 57 rows over 60 experts 18.5 -> 21.3).
  constexpr bool kOnce = kSource == kMxGroups || (kSource == kMxList && kEpi != kMxBf16);
  __shared__ floatx4 part[kSplit > 1 ? kMxWaves * kRT * 4 * kWave : 1];
  const int index = blockIdx.x / blocks, block = blockIdx.x - index * blocks;
  if constexpr (kSource == kMxGroups) {
    static_assert(kEpi == kMxBf16 && kRT == 2, "groups: bf16 rows, up to two row tiles");
    if (index == g.experts) {  // the rows of no group
      if (!g.zero_rest) return;
      const int first = min(max(g.bounds[0], 0), g.rows), last = min(max(g.bounds[g.experts], 0), g.rows);
      mx_zero_rows(g, make_int4(-1, 0, first, 0), block * kGroups * kMxRows, kGroups * kMxRows);
      mx_zero_rows(g, make_int4(-1, last, g.rows - last, 0), block * kGroups * kMxRows, kGroups * kMxRows);
      return;
    }
    const int end = min(max(g.bounds[index + 1], 0), g.rows);
    for (int at = min(max(g.bounds[index], 0), g.rows); at < end; at += 16 * kRT) {  // uniform
      const int4 item = make_int4(index, at, min(16 * kRT, end - at), 0);
      if (item.z > 16)
        mx_stream_item<2, kEpi, kSplit, kDirect, kOnce>(g, item, block, part);
      else
        mx_stream_item<1, kEpi, kSplit, kDirect, kOnce>(g, item, block, part);
      if (kSplit > 1) __syncthreads();  // `part` is read before the next tiles write it
    }
  } else if constexpr (kSource == kMxScan) {
    __shared__ MxScan scan;
    const int extra = mx_scan_extra(g.rows);
    int expert = index - extra, tile = 0;
    if (index < extra) {  // uniform
      mx_scan_further(g, index, scan);
      expert = scan.expert, tile = scan.tile;
      if (expert < 0) return;
    }
    const int count = mx_scan_pairs(g, expert, scan) - 16 * kRT * tile;
    static_assert(kRT == 1, "tiles of 16 pairs");
    if (count > 0)  // uniform
      mx_stream_item<kRT, kEpi, kSplit, kDirect, kOnce, true>(g, make_int4(expert, 16 * tile, min(16, count), 0), block,
                                                              part, scan.list);
  } else {
    int4 item;
    if constexpr (kSource == kMxPairs) {
      const int64_t expert = mx_pair_expert(g, index);
      if (expert < 0 || expert >= g.experts) return;  // uniform
      item = make_int4(static_cast<int>(expert), index, 1, 0);
    } else {
      item = mx_item(g, index, 16 * kRT);
      if (item.z <= 0) return;  // uniform
    }
    if (kEpi == kMxBf16 && item.x < 0) {
      mx_zero_rows(g, item, block * kGroups * kMxRows, kGroups * kMxRows);
      return;
    }
    mx_stream_item<kRT, kEpi, kSplit, kDirect, kOnce>(g, item, block, part);
  }
}

// Down product and combine of few rows in one launch: a workgroup owns one
// row and 64 outputs; its waves take the row's ranks in turn, each one row
// group of its expert's matrix times the rank's activations, and the ranks'
// fp32 results meet in LDS and are added in rank order.
constexpr int kMxMaxTopK = 16;
constexpr int kDownWaves = 8;
__global__ __launch_bounds__(kDownWaves * kWave) void mx_down_combine_kernel(MxGemm g, const void* __restrict__ weights,
                                                                     int weights_f32) {
  __shared__ float result[kMxMaxTopK][kMxRows];
  const int row = blockIdx.x / g.row_groups, rg = blockIdx.x - row * g.row_groups;
  const int lane = lane_id(), group = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (int r = wave; r < g.top_k; r += kDownWaves) {
    const int64_t pair = static_cast<int64_t>(row) * g.top_k + r;
    const int64_t expert = mx_pair_expert(g, pair);
    if (expert < 0 || expert >= g.experts) continue;
    // Every column of the MFMA's second operand is the pair's row; column 0 is kept.
    const uint8_t* codes = g.a + pair * g.steps * kMxOperandCodes + 16 * group;
    const uint8_t* scales = g.as + pair * g.steps * kMxOperandScales + 4 * (group & 1);
    const int64_t base = expert * g.row_groups + rg;
    const int32x4* w = reinterpret_cast<const int32x4*>(g.w + base * g.steps * kMxStepCodes) + lane;
    const uint2* ws = reinterpret_cast<const uint2*>(g.ws + base * g.steps * kMxStepScales) + lane;
    floatx4 acc[4] = {};
    for (int step = 0; step < g.steps; ++step) {
      int32x4 wf[2][4];
      const int32x4* wp = w + static_cast<int64_t>(step) * (kMxStepCodes / 16);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t) wf[h][t] = wp[(4 * h + t) * kWave];
      const uint2 wsc = ws[static_cast<int64_t>(step) * (kMxStepScales / 8)];
      const uint32_t sb = *reinterpret_cast<const uint32_t*>(scales + kMxOperandScales * step) >> (8 * (group >> 1));
      const int32x4* b = reinterpret_cast<const int32x4*>(codes + kMxOperandCodes * step);
      mfma_tiles<0>(wf[0], b[0], acc, wsc.x, sb);
      mfma_tiles<2>(wf[1], b[4], acc, wsc.y, sb);
    }
    if ((lane & 15) == 0) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *reinterpret_cast<floatx4*>(&result[r][32 * (t >> 1) + 8 * group + 4 * (t & 1)]) = acc[t];
    }
  }
  __syncthreads();
  if (threadIdx.x >= kMxRows) return;
  float sum = 0.0f;
  for (int r = 0; r < g.top_k; ++r) {
    const int64_t pair = static_cast<int64_t>(row) * g.top_k + r;
    const int64_t expert = mx_pair_expert(g, pair);
    if (expert >= 0 && expert < g.experts) sum = fmaf(route_weight(weights, weights_f32, pair), result[r][threadIdx.x], sum);
  }
  static_cast<uint16_t*>(g.out)[static_cast<int64_t>(row) * g.out_stride + kMxRows * rg + threadIdx.x] = f32_to_bf16(sum);
}

// Contraction-sized items (up to 128 rows).  A workgroup owns (item, 256
// weight rows); each of its four waves one row group of 64 and every row of
// the item, on the 32x32x64 MFMA (measured in registers alone 8.6 PFLOP/s with
// two waves a SIMD; the 16x16x128 one, whose operands are the same size for
// half the products, 6.2).  Weights go straight from memory into operands:
// the packed layout's 256-byte runs of 16 rows at one block serve both
// shapes.  The item's quantised rows are staged through a three-slot LDS ring,
// one step of 256 elements at a time: 128 bytes a row, its 16-byte part p at
// p ^ (row % 8), so that neither the stores (eight lanes a row) nor the reads
// (a lane a row) meet in a bank.  An item is multiplied in the smallest of
// four bodies (1 to 4 tiles of 32 rows) that holds it.
typedef float floatx16 __attribute__((ext_vector_type(16)));
constexpr int kMxTiledRows = 128;
constexpr int mx_slot_codes(int tiles) { return 32 * tiles * kMxOperandCodes; }
constexpr int mx_slot(int tiles) { return mx_slot_codes(tiles) + kMxThreads * 4; }  // (a word of scales a thread)
constexpr int kMxXcds = 8;
constexpr uint32_t kMxNowhere = 0xfffffff0u;  // an offset past every view

// f(integral_constant 0), .., f(integral_constant N - 1).
template <class F, int... I>
__device__ __forceinline__ void mx_each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void mx_each(F&& f) {
  mx_each_of(f, std::make_integer_sequence<int, N>{});
}

struct MxTiles {
  int n_tiles;  // 256-row weight tiles
  int run;      // consecutive items whose tiles one XCD takes together
  int item_rows;
};

template <int SA, int SB>
__device__ __forceinline__ floatx16 mfma_fp4_32(const int32x4& a, const int32x4& b, const floatx16& c, uint32_t sa,
                                                uint32_t sb) {
  const int32x8 av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  const int32x8 bv = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, kMxLow, kMxLow, SA, static_cast<int>(sa), SB,
                                                         static_cast<int>(sb));
}

// The sums of 32 rows for row group rg in the 32x32 output layout: lane half
// hl holds rows 8 j + 4 hl + i (element 4 j + i) of each 32-row half u of the
// group, columns 16 (j % 2) + 8 hl + 4 (j / 2) + i of it.
// Rows pass through the wave's own LDS, 144 bytes a row, so that a store
// writes eight whole 128-byte pieces instead of 32 bytes of 32 rows: a quarter
// of the lines to look up (4096 x 2048 x 1281, whose rows start anywhere in a
// line: 17.8 -> 13.6 us).
constexpr int kMxStoreRow = 2 * kMxRows + 16;
constexpr int kMxStoreArea = 32 * kMxStoreRow;
template <int kEpi>
__device__ __forceinline__ void mx_store32(const MxGemm& g, const floatx16 (&c)[2], int rg, const int4& item, int first,
                                           int count, const int32_t* targets, uint8_t* area) {
  const int lane = lane_id(), col = lane & 31, hl = lane >> 5;
  const int row = item.y + first + col;
  const bool live = first + col < count;
  if constexpr (kEpi == kMxAct) {
    float gate[16], up[16], v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = 4 * (i / 8 + 2 * (i / 4 % 2)) + i % 4;  // columns 16 (i / 8) + 8 hl + i % 8
      gate[i] = c[0][e];
      up[i] = c[1][e];
    }
    swiglu_values<16>(gate, up, v);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = MaxU32::apply(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    amax = MaxU32::apply(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32)));
    const uint32_t code = mx_scale_code(amax);
    const float inverse = mx_inverse(code);
    const uint32_t lo = mx_codes8(v, inverse), hi = mx_codes8(v + 8, inverse);
    if (!live) return;
    const uint32_t blocks = static_cast<uint32_t>(g.out_stride) / kMxBlock;
    const int64_t at = static_cast<int64_t>(row) * ((blocks + 7) / 8);  // in steps
    uint8_t* codes = static_cast<uint8_t*>(g.out) + at * kMxOperandCodes + rg * (kMxBlock / 2) + 4 * hl;
    *reinterpret_cast<uint32_t*>(codes) = lo;
    *reinterpret_cast<uint32_t*>(codes + 8) = hi;
    if (hl == 0) mx_operand_scale(g.out_scales + at * kMxOperandScales, rg, blocks, code);
  } else if constexpr (kEpi == kMxF32) {
    // A half of the group's columns at a time: 128 bytes a row, as above.
    const int part = lane & 7;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<floatx4*>(area + col * kMxStoreRow + 64 * (j % 2) + 32 * hl + 16 * (j / 2)) =
            floatx4{c[u][4 * j], c[u][4 * j + 1], c[u][4 * j + 2], c[u][4 * j + 3]};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 8 * k + (lane >> 3);
        const floatx4 w = *reinterpret_cast<const floatx4*>(area + r * kMxStoreRow + 16 * part);
        if (first + r < count)
          *reinterpret_cast<floatx4*>(static_cast<float*>(g.out) + static_cast<int64_t>(targets[first + r]) * g.out_stride +
                                      kMxRows * rg + 32 * u + 4 * part) = w;
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c[u][4 * j + 8 * (i / 4) + i % 4];
        *reinterpret_cast<int32x4*>(area + col * kMxStoreRow + 64 * u + 32 * j + 16 * hl) =
            __builtin_bit_cast(int32x4, mx_pack8(v));
      }
    const int part = lane & 7;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 8 * k + (lane >> 3);
      const MxWords4 w = __builtin_bit_cast(MxWords4, *reinterpret_cast<const int32x4*>(area + r * kMxStoreRow + 16 * part));
      if (first + r < count)
        mx_store16(static_cast<uint16_t*>(g.out) + static_cast<int64_t>(item.y + first + r) * g.out_stride,
                   kMxRows * rg + 8 * part, g.n, w, g.out_past);
    }
  }
}

template <int kRT, int kEpi, int kMax>
__device__ __forceinline__ void mx_tiled_body(const MxGemm& g, const int4& item, int n_tile, uint8_t* ring,
                                              int32_t* targets) {
  constexpr int kSlotCodes = mx_slot_codes(kMax), kSlot = mx_slot(kMax);
  const int tid = threadIdx.x, lane = lane_id(), col = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int rg = n_tile * kMxWaves + wave;
  const int rg_read = min(rg, g.row_groups - 1);
  const int count = min(item.z, 32 * kRT);
  const int steps = g.steps;

  // A thread stages part lane % 8 of rows 32 i + 8 wave + lane / 8, and four of
  // the eight scales of row tid / 2; rows past the item: its last row.  Offsets
  // are from the first quantised row (gathered rows; the host keeps them within
  // 32 bits) or from the item's first.
  const uint32_t pitch = static_cast<uint32_t>(steps) * kMxOperandCodes;
  const uint32_t scale_pitch = static_cast<uint32_t>(steps) * kMxOperandScales;
  constexpr bool kGather = kEpi == kMxAct;
  const int64_t first_row = kGather ? 0 : item.y;
  const int64_t view_rows = kGather ? g.a_rows : count;
  const __amdgpu_buffer_rsrc_t rows = BufferView(g.a + first_row * pitch, static_cast<uint32_t>(view_rows * pitch)).rsrc;
  const __amdgpu_buffer_rsrc_t row_scales =
      BufferView(g.as + first_row * scale_pitch, static_cast<uint32_t>(view_rows * scale_pitch)).rsrc;
  auto source_row = [&](int r) -> uint32_t {
    const int at = min(r, count - 1);
    return kGather ? static_cast<uint32_t>(g.sorted[item.y + at]) / static_cast<uint32_t>(g.top_k)
                   : static_cast<uint32_t>(at);
  };
  const int stage_row = 8 * wave + (lane >> 3), part = lane & 7;
  uint32_t src[kRT + 1];
#pragma unroll
  for (int i = 0; i < kRT; ++i) src[i] = source_row(32 * i + stage_row);
  src[kRT] = source_row(tid >> 1);
#pragma unroll
  for (int i = 0; i < kRT; ++i) src[i] = src[i] * pitch + 16 * part;
  src[kRT] = src[kRT] * scale_pitch + 4 * (tid & 1);
  const int stage_at = stage_row * kMxOperandCodes + 16 * (part ^ (stage_row & 7));

  // Weight operand (half u, slice q) of a step: row 32 u + col, block 2 q + hl,
  // which is tile 2 u + col / 16, half q / 2, group 2 (q % 2) + hl of the
  // packed layout; its scale is byte 2 u of `wsc[q]` once that lane's odd tiles
  // are shifted down.
  const int64_t base = (static_cast<int64_t>(item.x) * g.row_groups + rg_read) * steps;
  const __amdgpu_buffer_rsrc_t w = BufferView(g.w + base * kMxStepCodes, steps * kMxStepCodes).rsrc;
  const __amdgpu_buffer_rsrc_t ws = BufferView(g.ws + base * kMxStepScales, steps * kMxStepScales).rsrc;
  const int w_lane = (col >> 4) * 1024 + hl * 256 + (col & 15) * 16;
  const int ws_lane = (hl * 16 + (col & 15)) * 8;
  const int odd = 8 * (col >> 4);

  struct Rows {  // a step's rows on their way to LDS
    int32x4 codes[kRT];
    uint32_t scales;
  };
  int32x4 wf[4][2], operand[4];
  floatx2_hw wraw[2];
  uint32_t sb[kRT], sb_next[kRT], wsc[4];
  // Past the last step these read nothing: out of their views' range.
  auto load_weight = [&](int step, auto slice, auto half) {
    constexpr int q = decltype(slice)::value, u = decltype(half)::value;
    wf[q][u] = __builtin_amdgcn_raw_buffer_load_b128(
        w, w_lane + step * kMxStepCodes + (q / 2) * 4096 + (q % 2) * 512 + 2048 * u, 0, 0);
  };
  auto load_scales = [&](int step, auto index) {
    constexpr int i = decltype(index)::value;
    wraw[i] = __builtin_bit_cast(
        floatx2_hw, __builtin_amdgcn_raw_buffer_load_b64(ws, ws_lane + step * kMxStepScales + 256 * i, 0, 0));
  };
  auto load_row = [&](Rows& to, int step, auto index) {
    constexpr int i = decltype(index)::value;
    const bool live = step < steps;  // uniform
    if constexpr (i < kRT)
      to.codes[i] = __builtin_amdgcn_raw_buffer_load_b128(rows, live ? src[i] + step * kMxOperandCodes : kMxNowhere, 0, 0);
    else
      to.scales = __builtin_amdgcn_raw_buffer_load_b32(row_scales, live ? src[i] + step * kMxOperandScales : kMxNowhere, 0, 0);
  };
  auto store_rows = [&](uint8_t* slot, const Rows& from) {
#pragma unroll
    for (int i = 0; i < kRT; ++i)
      *reinterpret_cast<int32x4*>(slot + stage_at + 32 * i * kMxOperandCodes) = from.codes[i];
    *reinterpret_cast<uint32_t*>(slot + kSlotCodes + tid * 4) = from.scales;
  };
  auto read_operand = [&](const uint8_t* slot, auto unit) {
    constexpr int i = decltype(unit)::value, q = i / kRT, rt = i % kRT;
    operand[i % 4] = *reinterpret_cast<const int32x4*>(slot + (32 * rt + col) * kMxOperandCodes +
                                                       16 * ((2 * q + hl) ^ (col & 7)));
  };
  auto read_scale = [&](const uint8_t* slot, auto tile) {
    constexpr int rt = decltype(tile)::value;
    sb_next[rt] = *reinterpret_cast<const uint32_t*>(slot + kSlotCodes + (32 * rt + col) * kMxOperandScales + 4 * hl);
  };

  // Where the item's rows go, for the stores (written before the first barrier).
  if constexpr (kEpi == kMxF32)
    if (tid < 32 * kRT) targets[tid] = g.sorted[item.y + min(tid, count - 1)];

  floatx16 acc[kRT][2];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[rt][u][i] = 0.0f;

  // A step is 4 kRT units (slice, row tile) of one operand read and two
  // MFMAs, in this order and not the compiler's: the reads run kAhead units
  // ahead, across slices and into the next step; one load from memory goes
  // with each unit, a slice's weights once its registers are free, so that
  // loads that wait to be issued have MFMAs in flight before them.  Rows pass
  // through three slots: step s reads slot s % 3 and, in its last units, slot
  // (s + 1) % 3, which was stored in step s - 1 before the barrier in the
  // middle of step s; after that barrier nobody reads slot (s + 2) % 3, where
  // the rows of step s + 2 go, loaded since the middle of step s - 1.
  // (The barrier lies before the first read of the next slot.)
  constexpr int kUnits = 4 * kRT, kAhead = 3;
  constexpr int kBarrier = kUnits / 2 <= kUnits - kAhead ? kUnits / 2 : kUnits - kAhead;
  using std::integral_constant;
  Rows next;
  {
    Rows now;
    mx_each<kRT + 1>([&](auto i) { load_row(now, 0, i); });
    mx_each<2>([&](auto i) { load_scales(0, i); });
    mx_each<kRT + 1>([&](auto i) { load_row(next, 1, i); });
    mx_each<3>([&](auto q) {
      load_weight(0, q, integral_constant<int, 0>{});
      load_weight(0, q, integral_constant<int, 1>{});
    });
    store_rows(ring, now);
  }
  store_rows(ring + kSlot, next);
  mx_each<kRT + 1>([&](auto i) { load_row(next, 2, i); });
  lds_barrier();
  mx_each<kAhead>([&](auto i) { read_operand(ring, i); });
  mx_each<kRT>([&](auto i) { read_scale(ring, i); });
  const uint8_t* slot = ring;
  const uint8_t* slot_next = ring + kSlot;
  uint8_t* slot_free = ring + 2 * kSlot;
  for (int step = 0; step < steps; ++step) {
    wsc[0] = __float_as_uint(wraw[0][0]) >> odd, wsc[1] = __float_as_uint(wraw[1][0]) >> odd;
    wsc[2] = __float_as_uint(wraw[0][1]) >> odd, wsc[3] = __float_as_uint(wraw[1][1]) >> odd;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) sb[rt] = sb_next[rt];
    mx_each<kUnits>([&](auto unit) {
      constexpr int i = decltype(unit)::value, q = i / kRT, rt = i % kRT;
      if constexpr (i == kBarrier) {
        lds_barrier();
        store_rows(slot_free, next);
      }
      if constexpr (i + kAhead < kUnits)
        read_operand(slot, integral_constant<int, i + kAhead>{});
      else
        read_operand(slot_next, integral_constant<int, i + kAhead - kUnits>{});
      if constexpr (q == 2) read_scale(slot_next, integral_constant<int, rt>{});
      // this step's slice 3, then the next step's slices 0 to 2 as they end
      constexpr int kSlice = (q + 3) % 4;
      const int of = q == 0 ? step : step + 1;
      if constexpr (rt == 0) load_weight(of, integral_constant<int, kSlice>{}, integral_constant<int, 0>{});
      if constexpr (rt == (kRT > 1 ? 1 : 0))
        load_weight(of, integral_constant<int, kSlice>{}, integral_constant<int, 1>{});
      if constexpr (q == 1 && rt == kRT - 1) {
        load_scales(step + 1, integral_constant<int, 0>{});
        load_scales(step + 1, integral_constant<int, 1>{});
      }
      if constexpr (q == 2 && rt == kRT - 1) load_row(next, step + 3, integral_constant<int, kRT>{});
      if constexpr (q == 3) load_row(next, step + 3, integral_constant<int, rt>{});
      acc[rt][0] = mfma_fp4_32<0, q>(wf[q][0], operand[i % 4], acc[rt][0], wsc[q], sb[rt]);
      acc[rt][1] = mfma_fp4_32<2, q>(wf[q][1], operand[i % 4], acc[rt][1], wsc[q], sb[rt]);
      __builtin_amdgcn_sched_barrier(0);
    });
    const uint8_t* done = slot;
    slot = slot_next;
    slot_next = slot_free;
    slot_free = const_cast<uint8_t*>(done);
  }
  lds_barrier();
  if (rg >= g.row_groups) return;
  // Every wave has left the ring: its areas a wave's own (two that take turns,
  // where there is room).
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt)
    mx_store32<kEpi>(g, acc[rt], rg, item, 32 * rt, count, targets, ring + (kMax > 2 ? 2 * wave + rt % 2 : wave) * kMxStoreArea);
}

template <int kEpi, int kMax>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(kMax > 2 ? 2 : 3))) void mx_tiled_kernel(
    MxGemm g, MxTiles tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t ring[3 * mx_slot(kMax)];
  static_assert((kMax > 2 ? 2 : 1) * kMxWaves * kMxStoreArea <= 3 * mx_slot(kMax), "the waves' store areas fit the ring");
  __shared__ int32_t targets[kEpi == kMxF32 ? 32 * kMax : 1];
  // Runs of consecutive items go to the XCDs in turn (workgroup b runs on XCD
  // b % 8): a run's tiles share its rows, and an expert's consecutive items
  // its weights, in that XCD's L2.
  const int per_run = tiles.run * tiles.n_tiles;
  const int j = blockIdx.x / kMxXcds;
  const int in_run = j % per_run;
  const int index = ((j / per_run) * kMxXcds + blockIdx.x % kMxXcds) * tiles.run + in_run % tiles.run;
  const int n_tile = in_run / tiles.run;
  const int4 item = mx_item(g, index, tiles.item_rows);
  if (item.z <= 0) return;  // uniform
  if (kEpi == kMxBf16 && item.x < 0) {
    mx_zero_rows(g, item, n_tile * kMxWaves * kMxRows, kMxWaves * kMxRows);
    return;
  }
  if constexpr (kMax > 2) {
    if (item.z > 96) return mx_tiled_body<4, kEpi, kMax>(g, item, n_tile, ring, targets);
    if (item.z > 64) return mx_tiled_body<3, kEpi, kMax>(g, item, n_tile, ring, targets);
  }
  if (item.z > 32)
    mx_tiled_body<2, kEpi, kMax>(g, item, n_tile, ring, targets);
  else
    mx_tiled_body<1, kEpi, kMax>(g, item, n_tile, ring, targets);
}

// What a product needs first, in one launch: its rows quantised, and (by the
// first workgroup) its work items, from the groups' boundaries or from the
// routes' ids.
constexpr int kPrepareThreads = 1024;
enum MxPrepareWhat {
  kMxRowsOnly,
  kMxBounds,
  kMxRoutes,       // few enough pairs for one workgroup
  kMxRouteChunks,  // a workgroup per chunk of pairs counts, mx_place_kernel places
};
struct MxPrepare {
  MxQuantize rows;
  const int32_t* bounds;  // kMxBounds
  int groups;             // groups or experts
  int count;              // rows or (row, rank) pairs
  int zero_rest;
  const void* ids;  // kMxRoutes, kMxRouteChunks
  int ids_i64;
  int32_t* sorted;
  int chunks;
  int32_t* chunk_counts;  // [chunks][groups]
  int32_t* ranks;         // of a pair among its chunk's pairs of its expert
  int item_rows;
  int max_items;
  int4* items;
  int32_t* num_items;
};

// Boundaries lie on the device, where nobody has seen whether they ascend.  If
// they do not, groups share rows, and 65,536 of them may have more items than 31
// bits count (8,389,608 rows each: 32,768 times 65,544): items are counted up to that,
// which is past every list, instead of coming round to places before it.
__device__ __forceinline__ int mx_add_items(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

// Exclusive scan of the workgroup's pairs (rows, items) in place; returns the
// items' sum.  `sums` is LDS of one pair a wave, free again at the end.
__device__ __forceinline__ int mx_scan(int2* v, int2* sums) {
  const int wave = threadIdx.x / kWave, lane = lane_id();
  int2 scan = *v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int x = __shfl_up(scan.x, d), y = __shfl_up(scan.y, d);
    if (lane >= d) scan.x += x, scan.y = mx_add_items(scan.y, y);
  }
  if (lane == kWave - 1) sums[wave] = scan;
  __syncthreads();
  int2 before = make_int2(0, 0), all = before;
#pragma unroll
  for (int w = 0; w < kPrepareThreads / kWave; ++w) {
    if (w == wave) before = all;
    all.x += sums[w].x, all.y = mx_add_items(all.y, sums[w].y);
  }
  __syncthreads();
  v->x = before.x + scan.x - v->x;
  v->y = mx_add_items(before.y, scan.y) - v->y;
  return all.y;
}

// Every thread's group as items from `at` on (each of the workgroup's threads
// comes here): its first 16 by the thread, a busy group's others by the whole
// wave (16054 rows of one group, K 896 N 70: 30.0 us by its thread alone, 18.2
// so; but 1600 pairs over 60 experts, H384 I128: 31.2 us if only the first is the
// thread's, 19.9 so).
constexpr int kMxOwnItems = 16;
__device__ __forceinline__ void mx_write_items(const MxPrepare& p, int at, int expert, int first, int count) {
  const int lane = lane_id();
  auto write = [&](int i, int to, int e, int from, int n) {
    if (i * p.item_rows < n && i < p.max_items - to)
      p.items[to + i] = make_int4(e, from + i * p.item_rows, min(p.item_rows, n - i * p.item_rows), 0);
  };
  for (int i = 0; i < kMxOwnItems && i * p.item_rows < count; ++i) write(i, at, expert, first, count);
  for (uint64_t busy = __ballot(count > kMxOwnItems * p.item_rows); busy != 0; busy &= busy - 1) {
    const int of = __builtin_ctzll(busy);
    const int to = __shfl(at, of), e = __shfl(expert, of), from = __shfl(first, of), n = __shfl(count, of);
    const int items = min((n + p.item_rows - 1) / p.item_rows, p.max_items - to);
    for (int i = kMxOwnItems + lane; i < items; i += kWave) write(i, to, e, from, n);
  }
}

// Work items of ragged boundaries: group e's rows [b[e], b[e + 1]) in chunks
// of item_rows; with zero_rest the rows before b[0] and from b[E] on as items
// of expert -1.  Boundaries are clamped to [0, rows].
__device__ __forceinline__ void mx_items_of_bounds(const MxPrepare& p, int2* sums) {
  const int entries = p.groups + (p.zero_rest ? 2 : 0);
  auto bound = [&](int e) { return min(max(p.bounds[e], 0), p.count); };
  int base = 0;
  for (int from = 0; from < entries; from += kPrepareThreads) {
    const int e = from + threadIdx.x;
    int first = 0, last = 0, expert = -1;
    if (e < p.groups)
      first = bound(e), last = bound(e + 1), expert = e;
    else if (e == p.groups && e < entries)
      last = bound(0);
    else if (e < entries)
      first = bound(p.groups), last = p.count;
    const int count = max(last - first, 0);
    int2 at = make_int2(0, (count + p.item_rows - 1) / p.item_rows);
    const int total = mx_scan(&at, sums);
    mx_write_items(p, mx_add_items(base, at.y), expert, first, count);
    base = mx_add_items(base, total);
  }
  if (threadIdx.x == 0) *p.num_items = min(base, p.max_items);
}

// Routes grouped by expert: sorted[] holds the pairs of expert 0, 1, ..; ids
// that name no expert are left out.  A counting sort of one workgroup with
// LDS atomics: the order of an expert's pairs may differ from call to call,
// which no result depends on (a pair's row is multiplied by itself wherever it
// stands, and its results are stored by pair).  kBatch pairs a thread are
// loaded at once, so that up to 1024 kBatch pairs cost one round trip.
template <int kBatch>
__device__ __forceinline__ void mx_items_of_routes(const MxPrepare& p, int* cursor, int2* sums) {
  const int tid = threadIdx.x;
  int expert[kBatch];
  auto load = [&](int from) {
    int64_t id[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t at = min(from + j * kPrepareThreads + tid, p.count - 1);
      id[j] = p.ids_i64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at];
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      expert[j] = from + j * kPrepareThreads + tid < p.count && id[j] >= 0 && id[j] < p.groups ? static_cast<int>(id[j]) : -1;
  };
  constexpr int kRound = kPrepareThreads * kBatch;
  const bool once = p.count <= kRound;  // uniform
  if (tid < kMxMaxExperts) cursor[tid] = 0;
  load(0);
  __syncthreads();
  for (int from = 0; from < p.count; from += kRound) {
    if (from > 0) load(from);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (expert[j] >= 0) atomicAdd(&cursor[expert[j]], 1);
  }
  __syncthreads();
  const int count = tid < p.groups ? cursor[tid] : 0;
  int2 at = make_int2(count, (count + p.item_rows - 1) / p.item_rows);
  const int total = mx_scan(&at, sums);
  if (tid < p.groups) cursor[tid] = at.x;
  __syncthreads();
  mx_write_items(p, at.y, tid, at.x, count);
  if (tid == 0) *p.num_items = min(total, p.max_items);
  for (int from = 0; from < p.count; from += kRound) {
    if (!once) load(from);
    int place[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) place[j] = expert[j] >= 0 ? atomicAdd(&cursor[expert[j]], 1) : -1;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (place[j] >= 0) p.sorted[place[j]] = from + j * kPrepareThreads + tid;
  }
}

// The same spread over workgroups of kChunkPairs pairs, for batches whose LDS
// atomics one workgroup would be long at (29,344 pairs over 128 experts 26 us):
// each ranks its pairs and counts its experts' beside the rows' quantisation,
// then each sums the counts before its own and places its pairs.
constexpr int kChunkPairs = 2 * kPrepareThreads;
constexpr int kMxMaxChunks = 32;

__device__ __forceinline__ int mx_route_expert(const MxPrepare& p, int pair) {
  const int64_t at = min(pair, p.count - 1);
  const int64_t id = p.ids_i64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at];
  return pair < p.count && id >= 0 && id < p.groups ? static_cast<int>(id) : -1;
}

__device__ __forceinline__ void mx_count_chunk(const MxPrepare& p, int chunk, int* counts) {
  const int tid = threadIdx.x, first = chunk * kChunkPairs + tid;
  const int e0 = mx_route_expert(p, first), e1 = mx_route_expert(p, first + kPrepareThreads);
  if (tid < kMxMaxExperts) counts[tid] = 0;
  __syncthreads();
  if (e0 >= 0) p.ranks[first] = atomicAdd(&counts[e0], 1);
  if (e1 >= 0) p.ranks[first + kPrepareThreads] = atomicAdd(&counts[e1], 1);
  __syncthreads();
  if (tid < p.groups) p.chunk_counts[chunk * p.groups + tid] = counts[tid];
}

__global__ __launch_bounds__(kPrepareThreads) void mx_place_kernel(MxPrepare p) {
  __shared__ int place[kMxMaxExperts];
  __shared__ int2 sums[kPrepareThreads / kWave];
  const int tid = threadIdx.x, first = blockIdx.x * kChunkPairs + tid;
  int expert[2], rank[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int pair = first + j * kPrepareThreads;
    expert[j] = mx_route_expert(p, pair);
    rank[j] = p.ranks[min(pair, p.count - 1)];  // (of a pair of no expert: not used)
  }
  int all = 0, before = 0;
  if (tid < p.groups) {
#pragma unroll 8
    for (int c = 0; c < p.chunks; ++c) {
      const int n = p.chunk_counts[c * p.groups + tid];
      before += c < static_cast<int>(blockIdx.x) ? n : 0;
      all += n;
    }
  }
  int2 at = make_int2(all, (all + p.item_rows - 1) / p.item_rows);
  const int total = mx_scan(&at, sums);
  if (tid < p.groups) place[tid] = at.x + before;
  __syncthreads();
  if (blockIdx.x == 0) {
    mx_write_items(p, at.y, tid, at.x, all);
    if (tid == 0) *p.num_items = min(total, p.max_items);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (expert[j] >= 0) p.sorted[place[expert[j]] + rank[j]] = first + j * kPrepareThreads;
}

template <int kWhat, int kBatch = 1>
__global__ __launch_bounds__(kPrepareThreads) __attribute__((amdgpu_waves_per_eu(8))) void mx_prepare_kernel(MxPrepare p) {
  uint32_t block = blockIdx.x;
  if constexpr (kWhat != kMxRowsOnly) {
    __shared__ int cursor[kMxMaxExperts];
    __shared__ int2 sums[kPrepareThreads / kWave];
    const uint32_t others = kWhat == kMxRouteChunks ? p.chunks : 1;
    if (block < others) {
      if constexpr (kWhat == kMxBounds)
        mx_items_of_bounds(p, sums);
      else if constexpr (kWhat == kMxRoutes)
        mx_items_of_routes<kBatch>(p, cursor, sums);
      else
        mx_count_chunk(p, block, cursor);
      return;
    }
    block -= others;
  }
  mx_quantize_units<false, true, kPrepareThreads>(p.rows, block);
}

// out[t, :] = sum over ranks r of weights[t, r] * down[t * top_k + r, :] in
// rank order (fp32, one FMA a rank), rounded to bf16 once.  The down rows are
// fp32: they are summands that may cancel.  They are most of what the down
// product of a large batch writes and all that this kernel reads (29,344 pairs
// of 2048: 240 MB, read once at 5.5 TB/s; as scaled fp16 the whole call took 195
// us, so 222, but a result was no longer within fp32's error of its sum).  Ranks
// whose id names no expert add nothing (their down rows were never written).  A
// thread has four columns, so that a wave reads whole lines past the caches
// (eight: 222 -> 230); every rank's row piece is loaded before the first sum.
constexpr int kMxCombineColumns = kMxThreads * 4;
template <int kTopK>  // 0: any
__global__ __launch_bounds__(kMxThreads) void mx_combine_kernel(const float* __restrict__ down,
                                                                const void* __restrict__ ids, int ids_i64,
                                                                const void* __restrict__ weights, int weights_f32,
                                                                int any_top_k, int experts, int hidden, int slices,
                                                                uint16_t* __restrict__ out) {
  const int row = blockIdx.x / slices;
  const int column = (blockIdx.x % slices) * kMxCombineColumns + threadIdx.x * 4;
  if (column >= hidden) return;
  const int top_k = kTopK ? kTopK : any_top_k;
  const int64_t first = static_cast<int64_t>(row) * top_k;
  constexpr int kBatch = kTopK ? kTopK : 4;
  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int r0 = 0; r0 < top_k; r0 += kBatch) {
    floatx4 y[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      y[k] = __builtin_nontemporal_load(
          reinterpret_cast<const floatx4*>(down + (first + min(r0 + k, top_k - 1)) * hidden + column));
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int64_t pair = first + min(r0 + k, top_k - 1);
      const int64_t id = ids_i64 ? static_cast<const int64_t*>(ids)[pair] : static_cast<const int32_t*>(ids)[pair];
      const bool live = id >= 0 && id < experts && r0 + k < top_k;  // uniform
      const float w = route_weight(weights, weights_f32, pair);
      if (live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, y[k][i], acc[i]);
      }
    }
  }
  *reinterpret_cast<uint2*>(out + static_cast<int64_t>(row) * hidden + column) =
      make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
}

int mx_ceil(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

template <int kRT, int kEpi, bool kDirect, int kSource>
void launch_stream(const MxGemm& g, int items, hipStream_t s) {
  // Slices of the contraction: as many as there are steps, up to the waves.
  // (Eight waves and slices gain nothing: one row K 2048 N 1281 4.5 us either
  // way, one token's gate and up product 5.5 against 6.6.)
  const int split = g.steps >= 4 ? 4 : (g.steps >= 2 ? 2 : 1);
  const int blocks = mx_ceil(g.row_groups, kMxWaves / split);
  const dim3 grid(static_cast<unsigned>(items) * blocks), block(kMxThreads);
  if (split == 4)
    hipLaunchKernelGGL((mx_stream_kernel<kRT, kEpi, 4, kDirect, kSource>), grid, block, 0, s, g, blocks);
  else if (split == 2)
    hipLaunchKernelGGL((mx_stream_kernel<kRT, kEpi, 2, kDirect, kSource>), grid, block, 0, s, g, blocks);
  else
    hipLaunchKernelGGL((mx_stream_kernel<kRT, kEpi, 1, kDirect, kSource>), grid, block, 0, s, g, blocks);
}

// How a product runs: streaming (16 rows an item, or 32; the rows bf16 where
// they are at hand) or tiled (32, 64 or 128).
struct MxChoice {
  bool tiled;
  int item_rows;
};

template <int kEpi>
void launch_gemm(const MxGemm& g, MxChoice c, int items, hipStream_t s) {
  if (items <= 0) return;
  if (c.tiled) {
    // Runs of four items of one matrix where there are enough for every XCD
    // (8191 x 4096 x 4096 90.8 -> 87.3 us), else of two.
    const MxTiles tiles{mx_ceil(g.row_groups, kMxWaves), g.items == nullptr && items >= 8 * kMxXcds ? 4 : 2, c.item_rows};
    const int runs = mx_ceil(items, kMxXcds * tiles.run) * kMxXcds;
    const dim3 grid(static_cast<unsigned>(runs) * tiles.run * tiles.n_tiles), block(kMxThreads);
    if (c.item_rows > 64)
      hipLaunchKernelGGL((mx_tiled_kernel<kEpi, 4>), grid, block, 0, s, g, tiles);
    else
      hipLaunchKernelGGL((mx_tiled_kernel<kEpi, 2>), grid, block, 0, s, g, tiles);
  } else if constexpr (kEpi == kMxBf16) {
    if (c.item_rows <= 16)
      launch_stream<1, kEpi, true, kMxList>(g, items, s);
    else
      launch_stream<2, kEpi, true, kMxList>(g, items, s);
  } else {
    launch_stream<1, kEpi, kEpi == kMxAct, kMxList>(g, items, s);
  }
}

// Tiled items: as many rows as leave three quarters of the CUs a workgroup
// (`partial`: items that groups end early), for a larger item reads the weights
// less often.  Us at 32 / 64 / 128 rows an item, K and N 4096: 512 rows 19.5 /
// 19.5 / 23.7, 1024 rows 26.8 / 21.5 / 26.8, 2048 rows 49 / 35 / 30; K 2048 N
// 1281: 1024 rows 12.0 / 12.8 / 16.3, 4096 rows 22.4 / 20.4 / 20.1.
constexpr int kMxEnoughTiles = 192;
MxChoice choose_tiled(int64_t rows, int64_t partial, int64_t n) {
  const int64_t n_tiles = mx_ceil(n, kMxRows * kMxWaves);
  for (int item_rows = kMxTiledRows; item_rows > 32; item_rows /= 2)
    if (((rows + item_rows - 1) / item_rows + partial) * n_tiles >= kMxEnoughTiles) return {true, item_rows};
  return {true, 32};
}

int64_t stream_blocks(int64_t n, int64_t k) {
  const int64_t split = k > 3 * kMxStep ? 4 : (k > kMxStep ? 2 : 1);
  return mx_ceil(mx_ceil(n, kMxRows), kMxWaves / split);
}

// One matrix, every row: streaming while its workgroups are one round of the
// CUs.  Us, streaming 16 / 32 rows an item against tiled: K 2048 N 1281, 192
// rows 7.1 / 8.6 / 11.1, 384 rows 9.7 / 9.3 / 11.3, 512 rows 12.1 / 13.8 /
// 11.5; K and N 4096, 64 rows 8.9 / 12.0 / 16.6, 128 rows 13.9 / 12.7 / 17.3,
// 384 rows 33 / 29 / 18.5.
constexpr int kMxCus = 256;
MxChoice choose_linear(int64_t rows, int64_t n, int64_t k) {
  const int64_t blocks = stream_blocks(n, k);
  if (((rows + 15) / 16) * blocks <= kMxCus) return {false, 16};
  if (((rows + 31) / 32) * blocks <= kMxCus) return {false, 32};
  return choose_tiled(rows, 0, n);
}

// Rows grouped by expert: up to 8 rows an expert they stream, for more than one
// tile of 16 reads an expert's weights again.  Us a call in a graph, streaming /
// tiled: E256 H2048 I512, 8 rows an expert 90.8 / 100.2, 16 rows 127 / 108; E8
// H1920 I256, 164 rows an expert 31.5 / 26.0; E24 H128 I128, 500 rows an expert
// 33.7 / 26.8.
MxChoice choose_routed(int64_t pairs, int64_t experts, int64_t n) {
  const int64_t partial = (pairs < experts ? pairs : experts) / 2;
  return pairs <= 8 * experts ? MxChoice{false, 16} : choose_tiled(pairs, partial, n);
}

// Routes that need no sort (three launches, not four): few enough pairs for each
// workgroup to look through, and no more workgroups than four a CU, for they all
// do.  Us a call in a graph, without / with the sort: E16 H1024 I256, 160 / 480 /
// 1038 / 1184 pairs 11.6 / 15.7 / 20.1 / 21.4 against 15.6 / 17.8 / 20.0 / 20.7;
// E60 H640 I512, 456 pairs 17.9 against 21.3; E200 H512 I256, 800 pairs (992
// workgroups) 18.2 against 21.2; E16 H2048 I768, 320 pairs (1008) 25.0 against
// 24.2; but 560 pairs of it (1224) 28.7 against 25.0, E8 H1920 I512, 1280 pairs
// (1408) 41.1 against 26.9, and E256 H2048 I512, 512 pairs (4608) 80.5 against
// 73.2.
bool choose_scan(int64_t pairs, int64_t experts, int hidden, int inter) {
  if (pairs > kMxScanPairs) return false;
  const int64_t up = stream_blocks(2 * static_cast<int64_t>(inter), hidden), down = stream_blocks(hidden, inter);
  return (experts + mx_scan_extra(static_cast<int>(pairs))) * (up > down ? up : down) <= 4 * kMxCus;
}

// Byte arena of one call, carved in order at 256-byte boundaries.
struct Arena {
  uint8_t* base;
  int64_t used = 0;
  template <class T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
    return p;
  }
};

void set_weight(MxGemm& g, const uint8_t* w, const uint8_t* ws, int n, int k) {
  g.w = w, g.ws = ws, g.n = n;
  g.row_groups = mx_ceil(n, kMxRows), g.steps = mx_ceil(k, kMxStep), g.k_blocks = k / kMxBlock;
}

// A grouped product takes one of three ways:
//   walk     few rows, or few over many groups: one launch that walks each
//            group's row tiles and quantises them itself (no work items);
//   direct   few rows of one matrix: one launch that quantises them itself;
//   else     quantised rows, work items from the boundaries, the product.
// A group's workgroups walk its rows one tile after the other, so a busy group
// must be short.  Us, walked / not: one group of 21 rows K 768 N 584 8.8 / 12.3,
// of 48 K 2048 N 2048 10.6 / 11.9, of 64 13.9 / 12.0, of 160 28.2 / 12.1; 500
// rows over 16 groups 9.3 / 11.8 and, most of them in a few, 309 rows 20.6 / 12.5.
constexpr int kMxWalkRows = 512, kMxWalkAny = 48;
struct GroupedPlan {
  bool walk;
  MxChoice how;
  int max_items;
  uint8_t *q, *qs;
  int4* items;
  int32_t* num_items;
  int64_t bytes;
};

GroupedPlan plan_grouped(void* arena, int64_t rows, int experts, bool bounded, int n, int k) {
  GroupedPlan p{};
  p.walk = bounded && (rows <= kMxWalkAny || (rows <= kMxWalkRows && rows <= 16 * static_cast<int64_t>(experts)));
  if (p.walk) return p;
  const int64_t partial = rows < experts ? rows : experts;
  p.how = bounded ? choose_tiled(rows, partial / 2, n) : choose_linear(rows, n, k);
  // every group, and each of the two runs of rows in none, adds one partial item at most
  p.max_items = bounded ? static_cast<int>(rows / p.how.item_rows + (rows < experts + 2 ? rows : experts + 2))
                        : mx_ceil(rows, p.how.item_rows);
  if (!p.how.tiled) return p;
  Arena a{static_cast<uint8_t*>(arena)};
  p.q = a.take<uint8_t>(rows * mx_ceil(k, kMxStep) * kMxOperandCodes);
  p.qs = a.take<uint8_t>(rows * mx_ceil(k, kMxStep) * kMxOperandScales);
  if (bounded) {
    p.items = a.take<int4>(p.max_items);
    p.num_items = a.take<int32_t>(1);
  }
  p.bytes = a.used;
  return p;
}

MxQuantize operand_rows(const uint16_t* x, int64_t stride, int64_t rows, int k, uint8_t* codes, uint8_t* scales) {
  const uint32_t per_row = static_cast<uint32_t>(k) / 8;
  return {x, stride, static_cast<uint64_t>(rows) * per_row, per_row, mx_ceil(k, kMxStep), codes, scales};
}

int64_t prepare_blocks(const MxQuantize& q) {
  constexpr uint64_t kPerBlock = kPrepareThreads * kMxQuantizeUnits;
  return static_cast<int64_t>((q.units + kPerBlock - 1) / kPerBlock);
}

template <int kWhat, int kBatch = 1>
void launch_prepare(const MxPrepare& p, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL((mx_prepare_kernel<kWhat, kBatch>), dim3(blocks), dim3(kPrepareThreads), 0, s, p);
}

// Up to so many pairs each is an item of its own: us a call in a graph against
// grouped routes, E256 H2048 I512, 64 / 128 / 192 / 256 pairs 22.3 / 37.9 / 52.3 /
// 64.8 against 30.2 / 41.1 / 50.8 / 57.4; E128 I768, 64 / 128 / 192 pairs 31.2 /
// 47.5 / 65.2 against 36.4 / 46.8 / 54.1.  A few experts' pairs read the same
// weights again and again: past four workgroups a CU their experts' workgroups
// find them instead, if those are few enough (E8 H1536 I640, 32 / 64 / 128 pairs
// 14.6 / 17.4 / 22.8 against 13.7 / 14.2 / 15.2; E16 H1024 I256, 128 pairs 10.2
// against 11.3).  Where they are not, few wide experts, every pair streams its
// expert's weights for itself: by their bytes up to 16 times what E8 H4096 I14336
// needs at 128 pairs, which is neither timed nor avoided.
constexpr int kMxFewPairs = 128;
// Up to so many pairs are grouped by one workgroup, up to kMxMaxChunks chunks by
// a workgroup a chunk, more by the route sort over many workgroups.
constexpr int kMxOnePairs = 8 * kPrepareThreads;
struct MoePlan {
  bool few;   // no grouping, down product and combine in one launch
  bool scan;  // no grouping: every expert's workgroups find its pairs
  int chunks;  // 0: one workgroup groups the pairs; above kMxMaxChunks: the route sort
  MxChoice how;
  int max_items;
  int64_t pairs, scratch_ints;
  uint8_t *q, *qs, *act, *acts;
  float* rows;  // down rows
  int32_t *counts, *starts, *total, *sorted, *expert_ids, *num_items, *scratch;
  int4* items;
  int64_t bytes;
};

MoePlan plan_moe(void* arena, int64_t rows, int top_k, int experts, int hidden, int inter) {
  MoePlan p{};
  p.pairs = rows * top_k;
  p.chunks = p.pairs <= kMxOnePairs ? 0 : mx_ceil(p.pairs, kChunkPairs);
  p.scan = choose_scan(p.pairs, experts, hidden, inter);
  p.few = p.pairs <= kMxFewPairs && (!p.scan || p.pairs * stream_blocks(2 * static_cast<int64_t>(inter), hidden) <= 4 * kMxCus);
  p.scan = p.scan && !p.few;
  p.how = choose_routed(p.pairs, experts, 2 * static_cast<int64_t>(inter));
  p.max_items = d3_max_items(static_cast<int32_t>(p.pairs), experts, p.how.item_rows);
  Arena a{static_cast<uint8_t*>(arena)};
  const int64_t x_steps = mx_ceil(hidden, kMxStep), act_steps = mx_ceil(inter, kMxStep);
  p.act = a.take<uint8_t>(p.pairs * act_steps * kMxOperandCodes);
  p.acts = a.take<uint8_t>(p.pairs * act_steps * kMxOperandScales);
  if (!p.few) {
    if (p.how.tiled && !p.scan) {
      p.q = a.take<uint8_t>(rows * x_steps * kMxOperandCodes);
      p.qs = a.take<uint8_t>(rows * x_steps * kMxOperandScales);
    }
    p.rows = a.take<float>(p.pairs * hidden);
  }
  if (!p.few && !p.scan) {
    p.sorted = a.take<int32_t>(p.pairs);
    p.items = a.take<int4>(p.max_items);
    p.num_items = a.take<int32_t>(1);
    if (p.chunks > 0 && p.chunks <= kMxMaxChunks) {
      p.counts = a.take<int32_t>(static_cast<int64_t>(p.chunks) * experts);
      p.scratch = a.take<int32_t>(p.pairs);
    } else if (p.chunks > 0) {
      p.scratch_ints = d3_sort_wide_scratch_ints(static_cast<int32_t>(rows), top_k, experts);
      p.counts = a.take<int32_t>(experts);
      p.starts = a.take<int32_t>(experts);
      p.total = a.take<int32_t>(1);
      p.expert_ids = a.take<int32_t>(p.pairs);
      p.scratch = a.take<int32_t>(p.scratch_ints);
    }
  }
  p.bytes = a.used;
  return p;
}

// Widths whose offsets within a row group's weights and within an item's rows
// stay far inside the 32 bits of a buffer view, and the workgroups of a launch:
// a grid holds fewer than 2^32 threads.
constexpr int kMxMaxWidth = 1 << 20, kMxMaxColumns = 1 << 24;
constexpr int64_t kMxMaxWorkgroups = int64_t{1} << 24;

bool grouped_shape(int64_t rows, int experts, int n, int k) {
  return rows >= 0 && rows < (int64_t{1} << 30) && experts > 0 && experts <= (1 << 16) && n > 0 &&
         n <= kMxMaxColumns && k > 0 && k <= kMxMaxWidth && k % kGroup == 0;
}
bool moe_shape(int64_t rows, int top_k, int experts, int hidden, int inter) {
  return rows >= 0 && rows < (int64_t{1} << 26) && top_k >= 1 && top_k <= 16 && rows * top_k < (int64_t{1} << 26) &&
         experts >= 1 && experts <= 512 && hidden > 0 && inter > 0 && hidden <= kMxMaxWidth && inter <= kMxMaxWidth &&
         hidden % kGroup == 0 && inter % kGroup == 0;
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int64_t d3_mxfp4_grouped_workspace(int64_t rows, int32_t num_experts, int32_t bounded, int32_t n,
                                              int32_t k) {
  if (!grouped_shape(rows, num_experts, n, k)) return -1;
  return plan_grouped(nullptr, rows, num_experts, bounded != 0, n, k).bytes;
}

extern "C" int d3_mxfp4_grouped(const uint16_t* x, int64_t x_row_stride, int64_t rows, const int32_t* boundaries,
                                int32_t num_experts, const uint8_t* w, const uint8_t* ws, int32_t n, int32_t k,
                                uint16_t* out, int64_t out_row_stride, int32_t zero_rest, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  D3_REQUIRE(k > 0 && k % kGroup == 0, "mxfp4_grouped: K=%d must be a multiple of %d", k, kGroup);
  D3_REQUIRE(grouped_shape(rows, num_experts, n, k),
             "mxfp4_grouped: rows %lld (fewer than 2^30), experts %d (1 to 65536), N=%d (to 2^24), K=%d (to 2^20)",
             static_cast<long long>(rows), num_experts, n, k);
  D3_REQUIRE(boundaries != nullptr || num_experts == 1, "mxfp4_grouped: several experts need boundaries");
  D3_REQUIRE(rows == 0 || (x && w && ws && out), "mxfp4_grouped: null pointer");
  D3_REQUIRE(rows <= 1 || (x_row_stride >= 0 && out_row_stride >= n), "mxfp4_grouped: row strides");
  D3_REQUIRE(mx_aligned(x, 2) && mx_aligned(w, 16) && mx_aligned(ws, 8) && mx_aligned(out, 2) && mx_aligned(workspace, 16),
             "mxfp4_grouped: alignment");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  const GroupedPlan p = plan_grouped(workspace, rows, num_experts, boundaries != nullptr, n, k);
  D3_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes),
             "mxfp4_grouped: workspace of %lld bytes < required %lld", static_cast<long long>(workspace_bytes),
             static_cast<long long>(p.bytes));
  const int64_t most = p.walk ? num_experts + 1 : p.max_items;
  D3_SUPPORTED(most * mx_ceil(n, kMxRows) < kMxMaxWorkgroups, "mxfp4_grouped: more than 2^24 workgroups");
  // (rows of stride 0 need little memory: 2^25 of K 4096 would be 2^32 threads)
  D3_SUPPORTED(!p.how.tiled || prepare_blocks(operand_rows(x, x_row_stride, rows, k, p.q, p.qs)) + 1 <
                                   kMxMaxWorkgroups * kMxThreads / kPrepareThreads,
               "mxfp4_grouped: 2^37 elements of rows or more");
  hipStream_t s = as_stream(stream);
  MxGemm g{};
  set_weight(g, w, ws, n, k);
  g.a = p.q, g.as = p.qs, g.a_rows = rows, g.x = x, g.x_stride = x_row_stride, g.rows = static_cast<int>(rows);
  g.experts = num_experts, g.bounds = boundaries, g.zero_rest = zero_rest;
  g.out = out, g.out_stride = out_row_stride;
  // Results that the L2s do not hold leave them to the rows and weights: 8191 x
  // 4096 x 4096 87.5 -> 84.4 us and 16384 rows over 256 experts 82.5 -> 81.0 on
  // one card, 93 and 82.7 us either way on another.
  g.out_past = rows * static_cast<int64_t>(n) * 2 > (int64_t{1} << 25);
  if (p.walk) {
    launch_stream<2, kMxBf16, true, kMxGroups>(g, num_experts + 1, s);
    D3_LAUNCHED("mxfp4_grouped");
  }
  if (p.how.tiled) {
    MxPrepare prepare{};
    prepare.rows = operand_rows(x, x_row_stride, rows, k, p.q, p.qs);
    prepare.bounds = boundaries, prepare.groups = num_experts, prepare.count = static_cast<int>(rows);
    prepare.zero_rest = zero_rest, prepare.item_rows = p.how.item_rows, prepare.max_items = p.max_items;
    prepare.items = p.items, prepare.num_items = p.num_items;
    const unsigned blocks = static_cast<unsigned>(prepare_blocks(prepare.rows));
    if (boundaries != nullptr)
      launch_prepare<kMxBounds>(prepare, blocks + 1, s);
    else
      launch_prepare<kMxRowsOnly>(prepare, blocks, s);
    g.items = p.items, g.num_items = p.num_items, g.max_items = p.max_items;
  }
  launch_gemm<kMxBf16>(g, p.how, p.max_items, s);
  D3_LAUNCHED("mxfp4_grouped");
}

extern "C" int64_t d3_mxfp4_moe_workspace(int64_t rows, int32_t top_k, int32_t num_experts, int32_t hidden,
                                          int32_t intermediate) {
  if (!moe_shape(rows, top_k, num_experts, hidden, intermediate)) return -1;
  return plan_moe(nullptr, rows, top_k, num_experts, hidden, intermediate).bytes;
}

extern "C" int d3_mxfp4_moe(const uint16_t* x, int64_t x_row_stride, int64_t rows, const void* ids, int32_t ids_dtype,
                            const void* weights, int32_t weights_dtype, int32_t top_k, const uint8_t* w13,
                            const uint8_t* s13, const uint8_t* w2, const uint8_t* s2, int32_t num_experts,
                            int32_t hidden, int32_t intermediate, uint16_t* out, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  D3_REQUIRE(hidden > 0 && intermediate > 0 && hidden % kGroup == 0 && intermediate % kGroup == 0,
             "mxfp4_moe: hidden %d and intermediate %d must be multiples of %d", hidden, intermediate, kGroup);
  D3_REQUIRE(moe_shape(rows, top_k, num_experts, hidden, intermediate),
             "mxfp4_moe: rows %lld, top_k %d (1 to 16), experts %d (1 to 512), hidden %d and intermediate %d (to 2^20), "
             "fewer than 2^26 (row, rank) pairs",
             static_cast<long long>(rows), top_k, num_experts, hidden, intermediate);
  D3_REQUIRE(ids_dtype == D3_DTYPE_I32 || ids_dtype == D3_DTYPE_I64, "mxfp4_moe: ids must be int32 or int64");
  D3_REQUIRE(weights_dtype == D3_DTYPE_BF16 || weights_dtype == D3_DTYPE_F32, "mxfp4_moe: weights must be bf16 or f32");
  D3_REQUIRE(rows == 0 || (x && ids && weights && w13 && s13 && w2 && s2 && out && workspace), "mxfp4_moe: null pointer");
  D3_REQUIRE(rows <= 1 || x_row_stride >= 0, "mxfp4_moe: negative row stride");
  D3_REQUIRE(mx_aligned(x, 2) && mx_aligned(w13, 16) && mx_aligned(s13, 8) && mx_aligned(w2, 16) && mx_aligned(s2, 8) &&
                 mx_aligned(out, 16) && mx_aligned(workspace, 16) &&
                 mx_aligned(ids, ids_dtype == D3_DTYPE_I64 ? 8 : 4) &&
                 mx_aligned(weights, weights_dtype == D3_DTYPE_F32 ? 4 : 2),
             "mxfp4_moe: alignment");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  const MoePlan p = plan_moe(workspace, rows, top_k, num_experts, hidden, intermediate);
  D3_REQUIRE(workspace_bytes >= p.bytes, "mxfp4_moe: workspace of %lld bytes < required %lld",
             static_cast<long long>(workspace_bytes), static_cast<long long>(p.bytes));
  D3_SUPPORTED(rows * mx_ceil(hidden, kMxStep) * kMxOperandCodes < static_cast<int64_t>(kMxNowhere),
               "mxfp4_moe: more than 4 GiB of quantised rows");
  const int64_t widest = 2 * static_cast<int64_t>(intermediate) > hidden ? 2 * static_cast<int64_t>(intermediate) : hidden;
  D3_SUPPORTED(p.max_items * static_cast<int64_t>(mx_ceil(widest, kMxRows)) < kMxMaxWorkgroups &&
                   rows * mx_ceil(hidden, kMxCombineColumns) < kMxMaxWorkgroups,
               "mxfp4_moe: more than 2^24 workgroups");
  hipStream_t s = as_stream(stream);
  const int i64 = ids_dtype == D3_DTYPE_I64, f32 = weights_dtype == D3_DTYPE_F32;
  MxGemm up{}, down{};  // the two products
  set_weight(up, w13, s13, 2 * intermediate, hidden);
  up.x = x, up.x_stride = x_row_stride, up.a = p.q, up.as = p.qs, up.a_rows = rows;
  up.out = p.act, up.out_stride = intermediate, up.out_scales = p.acts;
  set_weight(down, w2, s2, hidden, intermediate);
  down.a = p.act, down.as = p.acts, down.out_stride = hidden;
  for (MxGemm* g : {&up, &down}) {
    g->items = p.items, g->num_items = p.num_items, g->max_items = p.max_items, g->sorted = p.sorted, g->top_k = top_k;
    g->ids = ids, g->ids_i64 = i64, g->experts = num_experts, g->rows = static_cast<int>(p.pairs);
  }
  if (p.few) {
    launch_stream<1, kMxAct, true, kMxPairs>(up, static_cast<int>(p.pairs), s);
    down.out = out;
    hipLaunchKernelGGL(mx_down_combine_kernel, dim3(static_cast<unsigned>(rows) * down.row_groups),
                       dim3(kDownWaves * kWave), 0, s, down, weights, f32);
    D3_LAUNCHED("mxfp4_moe");
  }
  const int slices = mx_ceil(hidden, kMxCombineColumns);
  const dim3 grid(static_cast<unsigned>(rows) * slices), block(kMxThreads);
  auto combine = [&] {
    auto kernel = top_k == 8 ? mx_combine_kernel<8> : mx_combine_kernel<0>;
    hipLaunchKernelGGL(kernel, grid, block, 0, s, p.rows, ids, i64, weights, f32, top_k, num_experts, hidden,
                       slices, out);
  };
  down.out = p.rows;
  if (p.scan) {
    const int items = num_experts + mx_scan_extra(static_cast<int>(p.pairs));
    launch_stream<1, kMxAct, true, kMxScan>(up, items, s);
    launch_stream<1, kMxF32, false, kMxScan>(down, items, s);
    combine();
    D3_LAUNCHED("mxfp4_moe");
  }
  MxPrepare prepare{};
  unsigned blocks = 0;
  if (p.how.tiled) {
    prepare.rows = operand_rows(x, x_row_stride, rows, hidden, p.q, p.qs);
    blocks = static_cast<unsigned>(prepare_blocks(prepare.rows));
  }
  if (p.chunks > kMxMaxChunks) {
    const int status = d3_sort_routes_wide(
        ids, ids_dtype, static_cast<int32_t>(rows), nullptr, top_k, num_experts, 1, p.counts, p.starts, p.total, p.sorted,
        p.expert_ids, static_cast<int32_t>(p.pairs), nullptr, p.how.item_rows, reinterpret_cast<int32_t*>(p.items),
        p.max_items, p.num_items, nullptr, p.scratch, p.scratch_ints, stream);
    if (status != D3_OK) return status;
    if (blocks > 0)
      launch_prepare<kMxRowsOnly>(prepare, blocks, s);
  } else {
    prepare.groups = num_experts, prepare.count = static_cast<int>(p.pairs);
    prepare.ids = ids, prepare.ids_i64 = i64, prepare.sorted = p.sorted;
    prepare.item_rows = p.how.item_rows, prepare.max_items = p.max_items;
    prepare.items = p.items, prepare.num_items = p.num_items;
    prepare.chunks = p.chunks, prepare.chunk_counts = p.counts, prepare.ranks = p.scratch;
    if (p.chunks > 0) {
      launch_prepare<kMxRouteChunks>(prepare, blocks + p.chunks, s);
      hipLaunchKernelGGL(mx_place_kernel, dim3(p.chunks), dim3(kPrepareThreads), 0, s, prepare);
    } else if (p.pairs <= kPrepareThreads) {
      launch_prepare<kMxRoutes, 1>(prepare, blocks + 1, s);
    } else {
      launch_prepare<kMxRoutes, 8>(prepare, blocks + 1, s);
    }
  }
  launch_gemm<kMxAct>(up, p.how, p.max_items, s);
  launch_gemm<kMxF32>(down, p.how, p.max_items, s);
  combine();
  D3_LAUNCHED("mxfp4_moe");
}
