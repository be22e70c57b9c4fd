// MXFP4 quantisation of rows, the way back, and the packed weight layout of
// the MXFP4 products.
//
// Both directions read and write every element once and are bound by HBM.
// bf16 tensors that no cache holds go past them: rows read from seven eighths of
// the 256 MiB last-level cache on, values written from half of it on.  Us, past /
// through the caches: rows of 98 MB 24.2 / 20.8, 197 MB 43.0 / 43.0 (38.1 where
// they are in the cache), 246 MB 52.5 / 57.2, 403 MB 82.9 / 90.9 (4.9 TB/s read,
// 6.2 with the codes written); values of 98 MB 20.5 / 21.1, 197 MB 37.8 / 40.6,
// 246 MB 46.4 / 57.7, 403 MB 74.1 / 91.4.
// fp32 ones never do: a lane's eight elements are two accesses of half its 32
// bytes, and past the caches nothing joins the halves of a line.  Rows of 49 MB
// 14.0 / 11.1, 403 MB 89.5 / 87.0; values of 154 MB 62 / 27.5, 403 MB 171 / 119.
#include "mxfp4.h"
#include "status.h"

namespace d3 {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowUnits = kMxQuantizeUnits;
constexpr int64_t kCachedIn = int64_t{7} << 25, kCachedOut = int64_t{1} << 27;

template <bool kF32, bool kOnce>
__global__ __launch_bounds__(kRowThreads) void quantize_kernel(MxQuantize q) {
  mx_quantize_units<kF32, false, kRowThreads, kOnce>(q, blockIdx.x);
}

template <bool kF32, bool kOnce>
__global__ __launch_bounds__(kRowThreads) void dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales, uint64_t units,
                                                                 void* __restrict__ out) {
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (kRowThreads * kRowUnits) + threadIdx.x;
  uint32_t word[kRowUnits], code[kRowUnits];
#pragma unroll
  for (int j = 0; j < kRowUnits; ++j) {
    const uint64_t u = first + static_cast<uint64_t>(j) * kRowThreads;
    const uint64_t at = u < units ? u : units - 1;
    word[j] = reinterpret_cast<const MxWord*>(codes)[at].w;
    code[j] = scales[at >> 2];
  }
#pragma unroll
  for (int j = 0; j < kRowUnits; ++j) {
    const uint64_t u = first + static_cast<uint64_t>(j) * kRowThreads;
    if (u >= units) return;
    const float scale = mx_scale(code[j]);
    float v[8];
    const floatx2_hw p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], 1.0f, 0);
    const floatx2_hw p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], 1.0f, 1);
    const floatx2_hw p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], 1.0f, 2);
    const floatx2_hw p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[j], 1.0f, 3);
    v[0] = p0[0] * scale, v[1] = p0[1] * scale, v[2] = p1[0] * scale, v[3] = p1[1] * scale;
    v[4] = p2[0] * scale, v[5] = p2[1] * scale, v[6] = p3[0] * scale, v[7] = p3[1] * scale;
    auto store = [&](int64_t at, MxVector4 w) {
      MxVector4* p = static_cast<MxVector4*>(out) + at;
      if constexpr (kOnce)
        __builtin_nontemporal_store(w, p);
      else
        *p = w;
    };
    if constexpr (kF32) {
      store(2 * u, __builtin_bit_cast(MxVector4, floatx4{v[0], v[1], v[2], v[3]}));
      store(2 * u + 1, __builtin_bit_cast(MxVector4, floatx4{v[4], v[5], v[6], v[7]}));
    } else {  // exact: a value has two significant bits and bf16 fp32's exponents
      store(u, MxVector4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7])});
    }
  }
}

// Weights [E, N, K / 2] codes and [E, N, K / 32] scales -> packed:
//   codes  [E][row groups][steps][half][tile][lane][16 bytes]: lane l holds
//          row l % 16 of the tile, elements 256 step + 128 half + 32 (l / 16)
//          .. + 32, an operand of the 16x16x128 MFMA: one wave load a tile
//          and half is 1 KiB of contiguous memory;
//   scales [E][row groups][steps][lane][8 bytes]: byte 4 half + tile, the
//          scale of that operand: a lane's scales of a step are one load, the
//          MFMA picks the byte.
// Padding (rows from N on, elements from K on) is zeros at scale 1.
__global__ __launch_bounds__(256) void pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                   int order, int n, int k, int row_groups, int steps,
                                                   uint64_t chunks, uint8_t* __restrict__ packed,
                                                   uint8_t* __restrict__ packed_scales) {
  const int kb_bytes = k / 2, k_blocks = k / kMxBlock;
  for (uint64_t c = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; c < chunks;
       c += static_cast<uint64_t>(gridDim.x) * 256) {
    const int lane = static_cast<int>(c % kWave);
    const int t = static_cast<int>(c / kWave % 4);
    const int half = static_cast<int>(c / (4 * kWave) % 2);
    const uint64_t block = c / (8 * kWave);  // (expert * row groups + row group) * steps + step
    const int step = static_cast<int>(block % steps);
    const uint64_t group = block / steps;
    const int rg = static_cast<int>(group % row_groups);
    const uint64_t expert = group / row_groups;
    const int row = mx_weight_row(order, n, rg, t, lane & 15);
    const int kblock = 8 * step + 4 * half + (lane >> 4);
    const bool live = row < n && kblock < k_blocks;
    const uint64_t at = expert * n + row;
    int4 v = make_int4(0, 0, 0, 0);
    uint8_t scale = 127;
    if (live) {
      v = *reinterpret_cast<const int4*>(codes + at * kb_bytes + 16 * kblock);
      scale = scales[at * k_blocks + kblock];
    }
    *reinterpret_cast<int4*>(packed + c * 16) = v;
    packed_scales[block * kMxStepScales + lane * 8 + 4 * half + t] = scale;
  }
}

constexpr int64_t kMaxUnits = int64_t{1} << 33;  // (a grid holds fewer than 2^32 threads)

unsigned row_blocks(uint64_t units) {
  return static_cast<unsigned>((units + kRowThreads * kRowUnits - 1) / (kRowThreads * kRowUnits));
}

}  // namespace

}  // namespace d3

using namespace d3;

extern "C" int d3_mxfp4_quantize(const void* x, int32_t x_dtype, int64_t x_row_stride, int64_t rows, int32_t width,
                                 uint8_t* codes, uint8_t* scales, void* stream) {
  D3_REQUIRE(rows >= 0 && width > 0 && width % kMxBlock == 0, "mxfp4_quantize: width %d must be a multiple of %d",
             width, kMxBlock);
  D3_REQUIRE(x_dtype == D3_DTYPE_BF16 || x_dtype == D3_DTYPE_F32, "mxfp4_quantize: x must be bf16 or f32");
  D3_REQUIRE(rows == 0 || (x && codes && scales), "mxfp4_quantize: null pointer");
  const bool f32 = x_dtype == D3_DTYPE_F32;
  D3_REQUIRE(rows <= 1 || x_row_stride >= 0, "mxfp4_quantize: negative row stride");
  D3_REQUIRE(mx_aligned(x, f32 ? 4 : 2), "mxfp4_quantize: x alignment");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  const uint32_t per_row = static_cast<uint32_t>(width) / 8;
  D3_SUPPORTED(rows <= kMaxUnits / per_row, "mxfp4_quantize: more than 2^36 elements");
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  const MxQuantize q{x, x_row_stride, units, per_row, 0, codes, scales};
  const dim3 grid(row_blocks(units)), block(kRowThreads);
  const bool once = rows * static_cast<int64_t>(width) * 2 > kCachedIn;
  auto kernel = f32 ? quantize_kernel<true, false> : (once ? quantize_kernel<false, true> : quantize_kernel<false, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), q);
  D3_LAUNCHED("mxfp4_quantize");
}

extern "C" int d3_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int32_t width,
                                   void* out, int32_t out_dtype, void* stream) {
  D3_REQUIRE(rows >= 0 && width > 0 && width % kMxBlock == 0, "mxfp4_dequantize: width %d must be a multiple of %d",
             width, kMxBlock);
  D3_REQUIRE(out_dtype == D3_DTYPE_BF16 || out_dtype == D3_DTYPE_F32, "mxfp4_dequantize: out must be bf16 or f32");
  D3_REQUIRE(rows == 0 || (codes && scales && out), "mxfp4_dequantize: null pointer");
  D3_REQUIRE(mx_aligned(out, 16), "mxfp4_dequantize: out must be 16-byte aligned");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  const uint32_t per_row = static_cast<uint32_t>(width) / 8;
  D3_SUPPORTED(rows <= kMaxUnits / per_row, "mxfp4_dequantize: more than 2^36 elements");
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  const dim3 grid(row_blocks(units)), block(kRowThreads);
  const bool f32 = out_dtype == D3_DTYPE_F32;
  const bool once = rows * static_cast<int64_t>(width) * 2 > kCachedOut;
  auto kernel =
      f32 ? dequantize_kernel<true, false> : (once ? dequantize_kernel<false, true> : dequantize_kernel<false, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), codes, scales, units, out);
  D3_LAUNCHED("mxfp4_dequantize");
}

extern "C" int d3_mxfp4_pack(const uint8_t* codes, const uint8_t* scales, int32_t num_experts, int32_t n, int32_t k,
                             int32_t order, uint8_t* packed, uint8_t* packed_scales, void* stream) {
  D3_REQUIRE(codes && scales && packed && packed_scales, "mxfp4_pack: null pointer");
  D3_REQUIRE(num_experts > 0 && n > 0 && k > 0 && k % kGroup == 0, "mxfp4_pack: K=%d must be a multiple of %d", k,
             kGroup);
  D3_REQUIRE(order == kMxOrderRows || order == kMxOrderGateUp, "mxfp4_pack: row order %d", order);
  D3_REQUIRE(order != kMxOrderGateUp || n % kMxRows == 0,
             "mxfp4_pack: gate and up need N=%d to be a multiple of %d", n, kMxRows);
  D3_REQUIRE(mx_aligned(codes, 16) && mx_aligned(packed, 16) && mx_aligned(packed_scales, 8),
             "mxfp4_pack: codes must be 16-byte aligned");
  const int row_groups = static_cast<int>((static_cast<int64_t>(n) + kMxRows - 1) / kMxRows);
  const int steps = static_cast<int>((static_cast<int64_t>(k) + kMxStep - 1) / kMxStep);
  const uint64_t chunks = static_cast<uint64_t>(num_experts) * row_groups * steps * (kMxStepCodes / 16);
  const uint64_t want = (chunks + 255) / 256;
  const unsigned blocks = static_cast<unsigned>(want < 65536 ? want : 65536);
  hipLaunchKernelGGL(pack_kernel, dim3(blocks), dim3(256), 0, as_stream(stream), codes, scales, order, n, k, row_groups,
                     steps, chunks, packed, packed_scales);
  D3_LAUNCHED("mxfp4_pack");
}

extern "C" int64_t d3_mxfp4_packed_bytes(int32_t num_experts, int32_t n, int32_t k, int32_t scales) {
  if (num_experts <= 0 || n <= 0 || k <= 0) return -1;
  const int64_t row_groups = (static_cast<int64_t>(n) + kMxRows - 1) / kMxRows;
  const int64_t steps = (static_cast<int64_t>(k) + kMxStep - 1) / kMxStep;
  return num_experts * row_groups * steps * (scales ? kMxStepScales : kMxStepCodes);
}
