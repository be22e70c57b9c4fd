// The kernel of batches whose tokens are all taken singly.
#include "paged_decode.h"

namespace d3 {
namespace {

constexpr int kWaves = 4;

template <int D, bool kE4m3>
__global__ __launch_bounds__(kWaves * kWave, 2) void paged_decode_kernel(PagedArgs a) {
  __shared__ DecodeShared<D, kWaves> shared;
  const int workgroup = static_cast<int>(blockIdx.x) / a.kv_heads;
  if (workgroup >= a.shares)
    paged_zero_rest(a, static_cast<int>(blockIdx.x) - a.shares * a.kv_heads, D);
  else
    decode_share<D, kE4m3, kWaves>(a, workgroup, static_cast<int>(blockIdx.x) % a.kv_heads, shared);
}

}  // namespace

void launch_paged_decode(const PagedArgs& a, int head_dim, bool e4m3, bool zero_rest, hipStream_t stream) {
  const unsigned workgroups = paged_workgroups(a, zero_rest);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(kWaves * kWave), 0, stream, a); };
  if (head_dim == 64)
    e4m3 ? run(paged_decode_kernel<64, true>) : run(paged_decode_kernel<64, false>);
  else if (head_dim == 128)
    e4m3 ? run(paged_decode_kernel<128, true>) : run(paged_decode_kernel<128, false>);
  else
    e4m3 ? run(paged_decode_kernel<256, true>) : run(paged_decode_kernel<256, false>);
}

}  // namespace d3
