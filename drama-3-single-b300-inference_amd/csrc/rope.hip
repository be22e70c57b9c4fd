// Rotary positions of packed rows, and appending keys and values to a paged
// cache with the rotation on the way.
//
// Pair i of a row at position p turns by p * turns[i] revolutions.  The product
// and its fraction are taken in fp64 (an fp32 product of a far position is off
// by a thousandth of a turn and more), sine and cosine of the remaining turn in
// fp32; the rotation is fp32, rounded once.
//
// Both calls read and write every element once and are bound by HBM; what a
// row costs besides is rotary_dim / 2 sines and cosines.  A workgroup takes as
// many rows as give each of its threads about one of them: they are computed
// once, held in LDS and used by all heads.  8191 x 40 x 128 bf16 rotated in 32 us (5.2
// TB/s of both directions; a copy moves 4.8); 8192 rows of 48 heads of 128 appended to an
// e4m3 cache in 39.5 us (4.7); one row 2.7 us, 64 appended 3.3: a launch.
#include "common.h"
#include "rows.h"
#include "status.h"

namespace d3 {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRowsHere = 8;     // rows of a workgroup
constexpr int64_t kCachedBytes = int64_t{32} << 20;  // the L2s together
constexpr int kMaxPairsHere = 512;  // sines and cosines in LDS
constexpr int kMaxColumns = 1 << 16;  // of a row: unit counts stay below what the division below is exact for

struct RopeTensor {  // [rows, heads, D], elements
  const void* in;
  int64_t in_row, in_head;
  void* out;
  int64_t out_row, out_head;
  int heads;
};

struct RopeArgs {
  RopeTensor q, k, v;  // q: rotated rows; k, v: to the cache (heads 0: none)
  int64_t rows;
  int head_dim, half;  // half = rotary_dim / 2
  int rotary_units, head_units;
  uint32_t head_units_inverse;  // 2^32 / head_units + 1: its high product divides exactly (counts below 2^16)
  int rows_here, slices;  // rows of a workgroup, workgroups of its units
  const double* turns;
  float magnitude;
  const void *positions, *row_slots;
  int positions_64, row_slots_64;
  // where k and v go
  int64_t k_page, k_token, v_page, v_token;
  const int32_t* page_table;
  int64_t table_stride, pages;
  int slots, max_pages, page_shift;
  const float *k_scales, *v_scales;
};

// x / scale rounded to e4m3, magnitudes above 448 to 448; NaN stays NaN.
__device__ __forceinline__ float e4m3_clamped(float x, float scale) {
  const float v = x / scale;
  return v > 448.0f ? 448.0f : (v < -448.0f ? -448.0f : v);
}

template <int V, typename T>
__device__ __forceinline__ void load_values(const void* p, float* v) {
  if constexpr (sizeof(T) == 2) {
    load_bf16<V>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = static_cast<const float*>(p)[i];
  }
}

// V values to fp32, bf16 or (kE4m3) codes of x / scale.
template <int V, typename T, bool kE4m3, bool kOnce>
__device__ __forceinline__ void store_values(void* p, const float* v, float scale) {
  if constexpr (kE4m3) {
    uint8_t* at = static_cast<uint8_t*>(p);
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamped(v[i], scale), e4m3_clamped(v[i + 1], scale), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamped(v[i + 2], scale), e4m3_clamped(v[i + 3], scale), w, true);
        *reinterpret_cast<int*>(at + i) = w;  // cache rows are 16-byte aligned, units whole words
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        at[i] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamped(v[i], scale), 0.0f, 0, false));
    }
  } else if constexpr (sizeof(T) == 2) {
    store_bf16<V, kOnce>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) static_cast<float*>(p)[i] = v[i];
  }
}

// One unit of a head: V pairs turned, or 2 V columns (the last unit perhaps V)
// that stay.  V columns are one access.
template <int V, typename T, bool kInterleaved, bool kE4m3, bool kOnce>
__device__ __forceinline__ void rope_unit(const RopeArgs& a, const T* in, void* out, int unit, bool turned,
                                          const float2* turn, float scale) {
  constexpr int kOut = kE4m3 ? 1 : static_cast<int>(sizeof(T));
  uint8_t* to = static_cast<uint8_t*>(out);
  float x[2 * V], y[2 * V];
  if (turned && unit < a.rotary_units) {
    const int first = kInterleaved ? 2 * V * unit : V * unit;
    const int second = kInterleaved ? first + V : first + a.half;
    load_values<V, T>(in + first, x);
    load_values<V, T>(in + second, x + V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 t = turn[V * unit + i];
      const int ia = kInterleaved ? 2 * i : i, ib = kInterleaved ? 2 * i + 1 : V + i;
      y[ia] = x[ia] * t.x - x[ib] * t.y;
      y[ib] = x[ia] * t.y + x[ib] * t.x;
    }
    store_values<V, T, kE4m3, kOnce>(to + first * kOut, y, scale);
    store_values<V, T, kE4m3, kOnce>(to + second * kOut, y + V, scale);
    return;
  }
  const int first = turned ? 2 * a.half + 2 * V * (unit - a.rotary_units) : 2 * V * unit;
  const bool both = first + 2 * V <= a.head_dim;
  if (first >= a.head_dim) return;
  load_values<V, T>(in + first, x);
  if (both) load_values<V, T>(in + first + V, x + V);
  store_values<V, T, kE4m3, kOnce>(to + first * kOut, x, scale);
  if (both) store_values<V, T, kE4m3, kOnce>(to + (first + V) * kOut, x + V, scale);
}

__device__ __forceinline__ int64_t index_at(const void* p, int is_64, int64_t i) {
  return is_64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

template <int V, typename T, bool kInterleaved, bool kE4m3, bool kAppend, bool kOnce>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
  __shared__ float2 turn[kMaxPairsHere];
  __shared__ int64_t place[kMaxRowsHere];  // page * page size + token, or -1
  const int64_t first = static_cast<int64_t>(blockIdx.x / a.slices) * a.rows_here;
  const int slice = static_cast<int>(blockIdx.x % a.slices);
  const int rows = static_cast<int>(a.rows - first < a.rows_here ? a.rows - first : a.rows_here);
  for (int i = threadIdx.x; i < rows * a.half; i += kRopeThreads) {
    const int r = i / a.half, pair = i - r * a.half;
    const double revolutions = static_cast<double>(index_at(a.positions, a.positions_64, first + r)) * a.turns[pair];
    float s, c;
    sincospif(2.0f * static_cast<float>(revolutions - rint(revolutions)), &s, &c);
    turn[i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  if constexpr (kAppend) {
    const int r = static_cast<int>(threadIdx.x);
    if (r < rows) {
      const int64_t position = index_at(a.positions, a.positions_64, first + r);
      const int64_t slot = index_at(a.row_slots, a.row_slots_64, first + r);
      int64_t at = -1;
      if (slot >= 0 && slot < a.slots && position >= 0 && (position >> a.page_shift) < a.max_pages) {
        const int64_t page = a.page_table[slot * a.table_stride + (position >> a.page_shift)];
        if (page >= 0 && page < a.pages) at = (page << a.page_shift) + (position & ((1 << a.page_shift) - 1));
      }
      place[r] = at;
    }
  }
  __syncthreads();
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int row_units = heads * a.head_units;
  for (int r = 0; r < rows; ++r) {
    const int64_t row = first + r;
    const float2* t = turn + r * a.half;
    for (int i = slice * kRopeThreads + static_cast<int>(threadIdx.x); i < row_units; i += a.slices * kRopeThreads) {
      int head = a.head_units == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), a.head_units_inverse));
      const int unit = i - head * a.head_units;
      if (head < a.q.heads) {
        rope_unit<V, T, kInterleaved, false, kOnce>(
            a, static_cast<const T*>(a.q.in) + row * a.q.in_row + head * a.q.in_head,
            static_cast<T*>(a.q.out) + row * a.q.out_row + head * a.q.out_head, unit, true, t, 1.0f);
        continue;
      }
      if constexpr (kAppend) {
        const int64_t at = place[r];
        if (at < 0) continue;
        head -= a.q.heads;
        const bool key = head < a.k.heads;
        if (!key) head -= a.k.heads;
        const RopeTensor& x = key ? a.k : a.v;
        const int64_t page = at >> a.page_shift, token = at & ((1 << a.page_shift) - 1);
        const int64_t to =
            page * (key ? a.k_page : a.v_page) + token * (key ? a.k_token : a.v_token) + head * x.out_head;
        const float* scales = key ? a.k_scales : a.v_scales;
        rope_unit<V, T, kInterleaved, kE4m3, kOnce>(
            a, static_cast<const T*>(x.in) + row * x.in_row + head * x.in_head,
            static_cast<uint8_t*>(x.out) + to * (kE4m3 ? 1 : static_cast<int>(sizeof(T))), unit, key, t,
            kE4m3 && scales != nullptr ? scales[head] : 1.0f);
      }
    }
  }
}

template <typename T, bool kE4m3, bool kAppend>
void launch_rope(RopeArgs a, int interleaved, hipStream_t stream) {
  // Columns of one access: 16 bytes where the head's parts are whole accesses
  // (rotated pairs in the half layout, whole units and what stays in both).
  const int rotary = 2 * a.half;
  auto fits = [&](int v) {
    return (interleaved ? rotary : a.half) % (interleaved ? 2 * v : v) == 0 && (a.head_dim - rotary) % v == 0 &&
           a.head_dim % v == 0;
  };
  constexpr int kWide = 16 / static_cast<int>(sizeof(T));
  const int v = fits(kWide) ? kWide : (fits(2) ? 2 : 1);
  a.rotary_units = a.half / v;
  a.head_units = a.rotary_units + (a.head_dim - rotary + 2 * v - 1) / (2 * v);
  const int all_units = (a.head_dim + 2 * v - 1) / (2 * v);  // of a value head, which nothing turns
  if (all_units > a.head_units) a.head_units = all_units;
  a.head_units_inverse = static_cast<uint32_t>((uint64_t{1} << 32) / a.head_units + 1);
  const int64_t units = static_cast<int64_t>(a.q.heads + a.k.heads + a.v.heads) * a.head_units;
  // Rows of a workgroup: about one sine and cosine a thread at most, three units a
  // thread (rope of 8191 x 40 x 128 31.7 us so, 33.0 with twice the rows; an e4m3
  // append of 8192 x 48 39.9 and 43.1; 3668 x 20 10.4 with three rows, 11.2 with one),
  // and no more than leave every CU four workgroups; few rows spread their units.
  int here = a.half ? kRopeThreads / a.half : kMaxRowsHere;
  const int64_t enough = (3 * kRopeThreads + units / 2) / units;
  if (here > enough) here = static_cast<int>(enough);
  if (here > a.rows / 1024) here = static_cast<int>(a.rows / 1024);
  // What the L2s cannot hold until its next reader is stored past them (38.2 -> 33.0 us
  // for those 8191 rows, 84 MB; smaller results stay).
  const bool once = v == kWide && sizeof(T) == 2 && a.rows * units * 2 * v * static_cast<int64_t>(sizeof(T)) > kCachedBytes;
  a.rows_here = here < 1 ? 1 : (here > kMaxRowsHere ? kMaxRowsHere : here);
  const int64_t groups = (a.rows + a.rows_here - 1) / a.rows_here;
  int64_t slices = groups >= 512 ? 1 : 512 / groups;
  const int64_t most = (units + kRopeThreads - 1) / kRopeThreads;
  a.slices = static_cast<int>(slices < most ? slices : most);
  const dim3 grid(static_cast<unsigned>(groups * a.slices)), block(kRopeThreads);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  auto with = [&](auto width, auto past) {
    constexpr int V = decltype(width)::value;
    constexpr bool kOnce = decltype(past)::value;
    if (interleaved)
      run(rope_kernel<V, T, true, kE4m3, kAppend, kOnce>);
    else
      run(rope_kernel<V, T, false, kE4m3, kAppend, kOnce>);
  };
  if (once) {
    if constexpr (sizeof(T) == 2) with(std::integral_constant<int, kWide>{}, std::true_type{});
  } else if (v == kWide) {
    with(std::integral_constant<int, kWide>{}, std::false_type{});
  } else if (v == 2) {
    with(std::integral_constant<int, 2>{}, std::false_type{});
  } else {
    with(std::integral_constant<int, 1>{}, std::false_type{});
  }
}

int check_rope(const char* name, const d3_rope* rope, int32_t head_dim) {
  D3_REQUIRE(rope->turns, "%s: null turns", name);
  D3_REQUIRE(rope->rotary_dim >= 2 && rope->rotary_dim % 2 == 0 && rope->rotary_dim <= head_dim,
             "%s: rotary width %d must be even and at most the head's %d", name, rope->rotary_dim, head_dim);
  D3_SUPPORTED(rope->rotary_dim <= 2 * kMaxPairsHere, "%s: rotary width above %d", name, 2 * kMaxPairsHere);
  return D3_OK;
}

bool is_index(int32_t dtype) { return dtype == D3_DTYPE_I32 || dtype == D3_DTYPE_I64; }

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_rope_rows(const void* x, int32_t x_dtype, int64_t x_row_stride, int64_t x_head_stride, int64_t rows,
                            int32_t heads, int32_t head_dim, const void* positions, int32_t positions_dtype,
                            const d3_rope* rope, void* out, int64_t out_row_stride, int64_t out_head_stride,
                            void* stream) {
  D3_REQUIRE(rope, "rope_rows: null rope");
  D3_REQUIRE(rows >= 0 && heads > 0 && head_dim > 0, "rope_rows: shape");
  D3_REQUIRE(x_dtype == D3_DTYPE_BF16 || x_dtype == D3_DTYPE_F32, "rope_rows: x must be bf16 or f32");
  D3_REQUIRE(is_index(positions_dtype), "rope_rows: positions must be int32 or int64");
  if (int status = check_rope("rope_rows", rope, head_dim)) return status;
  D3_SUPPORTED(static_cast<int64_t>(heads) * head_dim <= kMaxColumns, "rope_rows: more than %d columns a row", kMaxColumns);
  D3_SUPPORTED(rows < (int64_t{1} << 31) / 512, "rope_rows: more than 2^22 rows");
  D3_REQUIRE(rows == 0 || (x && positions && out), "rope_rows: null pointer");
  const bool f32 = x_dtype == D3_DTYPE_F32;
  D3_REQUIRE(aligned_to(x, f32 ? 4 : 2) && aligned_to(out, f32 ? 4 : 2), "rope_rows: alignment");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  RopeArgs a = {};
  a.q = {x, x_row_stride, x_head_stride, out, out_row_stride, out_head_stride, heads};
  a.rows = rows;
  a.head_dim = head_dim, a.half = rope->rotary_dim / 2;
  a.turns = rope->turns, a.magnitude = rope->magnitude;
  a.positions = positions, a.positions_64 = positions_dtype == D3_DTYPE_I64;
  if (f32)
    launch_rope<float, false, false>(a, rope->interleaved, as_stream(stream));
  else
    launch_rope<uint16_t, false, false>(a, rope->interleaved, as_stream(stream));
  D3_LAUNCHED("rope_rows");
}

extern "C" int d3_paged_append(const d3_paged_cache* cache, const uint16_t* k, int64_t k_row_stride,
                               int64_t k_head_stride, const uint16_t* v, int64_t v_row_stride, int64_t v_head_stride,
                               int64_t rows, const void* positions, int32_t positions_dtype, const void* row_slots,
                               int32_t row_slots_dtype, const d3_rope* rope, const uint16_t* q, int64_t q_row_stride,
                               int64_t q_head_stride, int32_t q_heads, uint16_t* q_out, int64_t q_out_row_stride,
                               int64_t q_out_head_stride, void* stream) {
  if (int status = check_paged_cache("paged_append", cache)) return status;
  const int32_t head_dim = cache->head_dim;
  D3_REQUIRE(rows >= 0 && q_heads >= 0, "paged_append: shape");
  D3_REQUIRE(is_index(positions_dtype) && is_index(row_slots_dtype),
             "paged_append: positions and row slots must be int32 or int64");
  if (rope)
    if (int status = check_rope("paged_append", rope, head_dim)) return status;
  D3_SUPPORTED((q_heads + 2 * static_cast<int64_t>(cache->kv_heads)) * head_dim <= kMaxColumns,
               "paged_append: more than %d columns a row", kMaxColumns);
  D3_SUPPORTED(rows < (int64_t{1} << 31) / 512, "paged_append: more than 2^22 rows");
  D3_REQUIRE(rows == 0 || (k && v && positions && row_slots), "paged_append: null pointer");
  D3_REQUIRE((q == nullptr) == (q_heads == 0) && (q == nullptr) == (q_out == nullptr),
             "paged_append: q, its heads and its result go together");
  if (rows == 0) {
    clear_error();
    return D3_OK;
  }
  RopeArgs a = {};
  a.q = {q, q_row_stride, q_head_stride, q_out, q_out_row_stride, q_out_head_stride, q_heads};
  a.k = {k, k_row_stride, k_head_stride, cache->keys, 0, cache->key_head_stride, cache->kv_heads};
  a.v = {v, v_row_stride, v_head_stride, cache->values, 0, cache->value_head_stride, cache->kv_heads};
  a.rows = rows;
  a.head_dim = head_dim;
  a.half = rope ? rope->rotary_dim / 2 : 0;
  a.turns = rope ? rope->turns : nullptr;
  a.magnitude = rope ? rope->magnitude : 1.0f;
  a.positions = positions, a.positions_64 = positions_dtype == D3_DTYPE_I64;
  a.row_slots = row_slots, a.row_slots_64 = row_slots_dtype == D3_DTYPE_I64;
  a.k_page = cache->key_page_stride, a.k_token = cache->key_token_stride;
  a.v_page = cache->value_page_stride, a.v_token = cache->value_token_stride;
  a.page_table = cache->page_table, a.table_stride = cache->table_stride;
  a.pages = cache->pages, a.slots = cache->slots, a.max_pages = cache->max_pages;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(cache->page_size));
  a.k_scales = cache->key_scales, a.v_scales = cache->value_scales;
  const int interleaved = rope ? rope->interleaved : 0;
  if (cache->dtype == D3_DTYPE_E4M3)
    launch_rope<uint16_t, true, true>(a, interleaved, as_stream(stream));
  else
    launch_rope<uint16_t, false, true>(a, interleaved, as_stream(stream));
  D3_LAUNCHED("paged_append");
}
