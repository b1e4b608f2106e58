// The range of block scales. Shared by the block quantizer, which marks its tiles, and
// the grouped GEMM, which reads the marks.
#pragma once

#include "common.cuh"

namespace aqtb200 {

constexpr float SCALE_MAX_FLOAT = 0x1.fffffep127f;

__device__ __forceinline__ bool finite_nonzero(float x) { return x != 0.f && fabsf(x) <= SCALE_MAX_FLOAT; }

// The product of two scales within 2^-63 .. 2^63 is a normal f32 number, and a block's
// sum times either of them too. Others have to be looked at together.
__device__ __forceinline__ bool may_be_far(float x) {
  return finite_nonzero(x) && (fabsf(x) < 0x1p-63f || fabsf(x) > 0x1p63f);
}

}  // namespace aqtb200
