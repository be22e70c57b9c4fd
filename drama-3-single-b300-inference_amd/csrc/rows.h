// What the attention operators share: bf16 rows in memory at any alignment of
// their elements, and the checks of a paged cache.
#pragma once

#include "common.h"
#include "status.h"

namespace d3 {

inline bool aligned_to(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// gfx950 takes wide accesses at any address: odd row strides cost no narrow path.
typedef uint32_t RowVector4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t RowWord __attribute__((aligned(2)));

// N bf16 values (8, 2 or 1) to fp32, and N fp32 values rounded to bf16.
template <int N>
__device__ __forceinline__ void load_bf16(const void* p, float* v) {
  static_assert(N == 8 || N == 2 || N == 1, "one access");
  if constexpr (N == 8) {
    const RowVector4 w = *static_cast<const RowVector4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
  } else if constexpr (N == 2) {
    const uint32_t w = *static_cast<const RowWord*>(p);
    v[0] = bf16_lo(w), v[1] = bf16_hi(w);
  } else {
    v[0] = bf16_to_f32(*static_cast<const uint16_t*>(p));
  }
}
// (kOnce: eight values past the L2s.)
template <int N, bool kOnce = false>
__device__ __forceinline__ void store_bf16(void* p, const float* v) {
  if constexpr (N == 8) {
    const RowVector4 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    if constexpr (kOnce)
      __builtin_nontemporal_store(w, static_cast<RowVector4*>(p));
    else
      *static_cast<RowVector4*>(p) = w;
  } else if constexpr (N == 2) {
    *static_cast<RowWord*>(p) = pack_bf16x2(v[0], v[1]);
  } else {
    *static_cast<uint16_t*>(p) = f32_to_bf16(v[0]);
  }
}

// A cache the kernels can walk: sizes that say what the pointers hold, rows of whole 16-byte parts.
inline int check_paged_cache(const char* name, const d3_paged_cache* c) {
  D3_REQUIRE(c, "%s: null cache", name);
  D3_REQUIRE(c->dtype == D3_DTYPE_BF16 || c->dtype == D3_DTYPE_E4M3, "%s: a cache is bf16 or e4m3", name);
  D3_REQUIRE(c->kv_heads > 0 && c->head_dim > 0 && c->pages > 0 && c->slots > 0 && c->max_pages > 0,
             "%s: cache shape", name);
  D3_REQUIRE(c->page_size > 0 && (c->page_size & (c->page_size - 1)) == 0, "%s: page size %d must be a power of two",
             name, c->page_size);
  D3_SUPPORTED(c->pages < (int64_t{1} << 31), "%s: more than 2^31 pages", name);
  D3_SUPPORTED(static_cast<int64_t>(c->max_pages) * c->page_size <= (int64_t{1} << 30),
               "%s: slots of more than 2^30 tokens", name);
  for (const int64_t stride : {c->key_page_stride, c->key_head_stride, c->key_token_stride, c->value_page_stride,
                               c->value_head_stride, c->value_token_stride})
    D3_SUPPORTED(stride >= 0 && stride < (int64_t{1} << 31), "%s: a stride of 2^31 elements and more", name);
  D3_REQUIRE(c->keys && c->values && c->page_table, "%s: null cache pointer", name);
  const int64_t part = c->dtype == D3_DTYPE_BF16 ? 8 : 16;
  D3_REQUIRE(aligned_to(c->keys, 16) && aligned_to(c->values, 16), "%s: cache alignment", name);
  D3_REQUIRE(c->head_dim % part == 0 && c->key_page_stride % part == 0 && c->key_head_stride % part == 0 &&
                 c->key_token_stride % part == 0 && c->value_page_stride % part == 0 &&
                 c->value_head_stride % part == 0 && c->value_token_stride % part == 0,
             "%s: cache rows and strides must be multiples of 16 bytes", name);
  return D3_OK;
}

}  // namespace d3
