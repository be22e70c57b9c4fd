// MXFP4 building blocks (OCP Microscaling Formats): e2m1 codes, two a byte
// with the even element in the low nibble, and one e8m0 scale (a power of
// two, code - 127 its exponent, code 255 NaN) per 32 elements of a row.
#pragma once

#include "common.h"
#include "expert_tile.h"

namespace d3 {

constexpr int kMxBlock = 32;       // elements per scale
constexpr int kMxRows = 64;        // weight rows of a packed row group (four 16-row MFMA tiles)
constexpr int kMxStep = 256;       // contracted elements of a packed step (two MFMAs deep)
constexpr int kMxStepCodes = kMxRows * kMxStep / 2;          // 8 KiB of codes per row group and step
constexpr int kMxStepScales = kMxRows * kMxStep / kMxBlock;  // 512 bytes of scales
constexpr int kMxOperandCodes = kMxStep / 2;         // a quantised row's codes per step
constexpr int kMxOperandScales = kMxStep / kMxBlock;  // and scales
constexpr int kMxLow = 4;  // the MFMA's format code of e2m1 operands

inline bool mx_aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Row orders of a packed weight: which row of W row m = 4 g + i (i < 4) of
// tile t of a row group holds.  The MFMAs' output lanes hold rows 4 g + i of
// every tile; with these orders a pair of tiles is eight consecutive columns.
constexpr int kMxOrderRows = 0;    // 32 (t / 2) + 8 g + 4 (t % 2) + i
constexpr int kMxOrderGateUp = 1;  // tiles 0-1 gate, 2-3 up rows 32 rg + 8 g + 4 (t % 2) + i: a lane holds both

// Row of W that row m of tile t of row group rg holds; rows from n on are padding.
__host__ __device__ __forceinline__ int mx_weight_row(int order, int n, int rg, int t, int m) {
  const int in_pair = 8 * (m >> 2) + 4 * (t & 1) + (m & 3);
  if (order == kMxOrderRows) return kMxRows * rg + 32 * (t >> 1) + in_pair;
  return (t >= 2 ? n / 2 : 0) + 32 * rg + in_pair;
}

// Quantised rows as the products read them: codes in row order at a pitch of
// whole steps, scales per step as byte 4 (block % 2) + block / 2 of its 8
// blocks: a lane of the 32x32x64 MFMA (block % 2 is its half of the wave) finds
// the scales of a step's four MFMAs in one word, one of the 16x16x128 MFMA
// (block % 4 is its group) both of its scales in one word, two bytes apart.
// A row whose width is an odd multiple of 128 has its last half step's scales
// zeroed here (the weights' codes are zeros there, the row's are whatever the
// buffer holds: no e2m1 code is an infinity or a NaN, but scale 255 would be).
__device__ __forceinline__ void mx_operand_scale(uint8_t* row, uint32_t block, uint32_t blocks, uint32_t code) {
  const uint32_t step = block >> 3;
  uint8_t* at = row + step * kMxOperandScales + 4 * (block & 1) + ((block & 7) >> 1);
  *at = static_cast<uint8_t>(code);
  if (8 * step + 4 >= blocks) at[2] = 0;  // the last step's second half is padding
}

// Scale code of a block whose largest magnitude has the fp32 bits `amax`
// (sign bit clear): floor(log2 amax) - 2, so that the largest element lies in
// [4, 8) scaled; 0 (2^-127) for zero blocks and those below 2^-124; 255 (NaN)
// where an element is infinite or NaN, which the whole block then stands for.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e >= 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// 2^(127 - code), the reciprocal of a scale: exact for every code of
// mx_scale_code (0 .. 252); 0 for 255, whose codes are then zeros.
__device__ __forceinline__ float mx_inverse(uint32_t code) {
  return code == 255u ? 0.0f : __uint_as_float((254u - code) << 23);
}

// Eight scaled values (magnitudes below 8) as e2m1 codes, v[0] in the low
// nibble: the gfx950 conversion at scale 1, round to nearest even, above 6 to
// 6.  The product by a power of two is exact (fp32 subnormals are kept), so
// one rounding is made.  A block at scale NaN gets zero codes.
__device__ __forceinline__ uint32_t mx_codes8(const float* v, float inverse) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = v[i] * inverse;
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, s[0], s[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[2], s[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[4], s[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[6], s[7], 1.0f, 3);
  return inverse == 0.0f ? 0u : w;
}

// 2^(code - 127): a subnormal for code 0, NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fc00000u : (code ? code << 23 : 0x00400000u));
}

typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));

// Largest magnitude of bf16 pairs as bf16 bits in each half.
template <int N>
__device__ __forceinline__ uint16x2 mx_amax_bf16(const uint32_t* w) {
  uint16x2 amax = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) amax = __builtin_elementwise_max(amax, __builtin_bit_cast(uint16x2, w[i] & 0x7fff7fffu));
  return amax;
}

// mx_codes8 of four words of bf16 pairs: the conversion divides by the scale
// itself (the same codes for every bf16 value and every scale, 2^-127
// included: compared on the device).
__device__ __forceinline__ uint32_t mx_codes8_bf16(const uint32_t* w, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
}

// Memory words at the alignment of their elements only: gfx950 takes wide
// accesses at any address, so odd row strides cost no narrow path.
struct __attribute__((packed, aligned(2))) MxWords4 { uint32_t w[4]; };
struct __attribute__((packed, aligned(1))) MxWord { uint32_t w; };
typedef uint32_t MxVector4 __attribute__((ext_vector_type(4), aligned(2)));

// Rows -> codes: a lane takes 8 consecutive elements, four lanes a block of
// 32.  The block's largest magnitude is an integer maximum of the values' bits
// (which orders NaN above infinity above every number), exchanged inside the
// quad with two DPP moves.  kOperand: the layout the products read, `steps`
// steps a row; else plain rows.
struct MxQuantize {
  const void* x;
  int64_t stride;
  uint64_t units;    // of 8 elements
  uint32_t per_row;  // units a row
  int steps;
  uint8_t* codes;
  uint8_t* scales;
};
constexpr int kMxQuantizeUnits = 4;  // units a thread has in flight

__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  v = MaxU32::apply(v, dpp_move<kDppQuad1032>(v, 0u));
  return MaxU32::apply(v, dpp_move<kDppQuad2301>(v, 0u));
}

// kOnce: the rows are larger than the caches and loaded non-temporally.
template <bool kF32, bool kOperand, int kThreads, bool kOnce = false>
__device__ __forceinline__ void mx_quantize_units(const MxQuantize& q, uint32_t block) {
  constexpr int kUnits = kMxQuantizeUnits;
  const uint64_t first = static_cast<uint64_t>(block) * (kThreads * kUnits) + threadIdx.x;
  MxWords4 raw[kUnits][kF32 ? 2 : 1];
  uint64_t row[kUnits];
  uint32_t unit[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const uint64_t u = first + static_cast<uint64_t>(j) * kThreads;
    const uint64_t at = u < q.units ? u : q.units - 1;
    row[j] = (at >> 32) == 0 ? static_cast<uint32_t>(at) / q.per_row : at / q.per_row;
    unit[j] = static_cast<uint32_t>(at - row[j] * q.per_row);
    const int64_t element = static_cast<int64_t>(row[j]) * q.stride + 8 * static_cast<int64_t>(unit[j]);
    const MxVector4* p = reinterpret_cast<const MxVector4*>(static_cast<const uint8_t*>(q.x) + element * (kF32 ? 4 : 2));
#pragma unroll
    for (int h = 0; h < (kF32 ? 2 : 1); ++h) {
      const MxVector4 v = kOnce ? __builtin_nontemporal_load(p + h) : p[h];
      raw[j][h] = __builtin_bit_cast(MxWords4, v);
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const uint64_t u = first + static_cast<uint64_t>(j) * kThreads;
    uint32_t code, word;
    if constexpr (kF32) {
      float v[8];
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = __uint_as_float(raw[j][i / 4].w[i % 4]);
        amax = MaxU32::apply(amax, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      code = mx_scale_code(mx_quad_max(amax));
      word = mx_codes8(v, mx_inverse(code));
    } else {
      const uint16x2 amax = mx_amax_bf16<4>(raw[j][0].w);
      code = mx_scale_code(mx_quad_max(MaxU32::apply(amax[0], amax[1])) << 16);
      word = mx_codes8_bf16(raw[j][0].w, mx_scale(code));
      if (code == 255u) word = 0;
    }
    if (u >= q.units) continue;
    if constexpr (kOperand) {
      *reinterpret_cast<uint32_t*>(q.codes + row[j] * q.steps * kMxOperandCodes + 4 * static_cast<uint64_t>(unit[j])) =
          word;
      if ((unit[j] & 3) == 0)
        mx_operand_scale(q.scales + row[j] * q.steps * kMxOperandScales, unit[j] >> 2, q.per_row >> 2, code);
    } else {
      reinterpret_cast<MxWord*>(q.codes)[u].w = word;
      if ((u & 3) == 0) q.scales[u >> 2] = static_cast<uint8_t>(code);
    }
  }
}

}  // namespace d3
