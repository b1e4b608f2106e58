// Row groups given by their sizes on the device (rows of one expert, one after
// the other). Shared by the block quantizer and the grouped GEMM.
#pragma once

#include "common.cuh"

namespace aqtb200 {

// Size of group g, made safe: negative sizes count as zero, and callers cut the
// running sum at the number of rows that exist.
__device__ __forceinline__ int64_t group_size_at(const void* sizes, int is64, int64_t g) {
  const int64_t v = is64 ? __ldg((const long long*)sizes + g) : (int64_t)__ldg((const int*)sizes + g);
  return v < 0 ? 0 : v;
}

// Inclusive prefix sum over the warp.
__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

}  // namespace aqtb200
