// The range of block scales. Shared by the block quantizer, which notes it for each of
// its tiles, and the grouped GEMM, which reads the notes.
#pragma once

#include "common.cuh"

namespace aqtb200 {

constexpr float SCALE_MAX_FLOAT = 0x1.fffffep127f, SCALE_MIN_NORMAL = 0x1p-126f;

__device__ __forceinline__ bool finite_nonzero(float x) { return x != 0.f && fabsf(x) <= SCALE_MAX_FLOAT; }

// A note on 128 x 128 elements: sixteen bytes, two from each of eight warps -- 255 less
// the smallest exponent of its finite scales, and the largest; zeros without any -- so
// that notes are joined by the larger of each byte.
__device__ __forceinline__ uint16_t scale_note(float s) {  // of a warp; a lane without one: 0
  const uint32_t e = finite_nonzero(s) ? (__float_as_uint(s) >> 23) & 255u : 0u;
  const uint32_t lo = __reduce_max_sync(0xffffffffu, e ? 255u - e : 0u);
  const uint32_t hi = __reduce_max_sync(0xffffffffu, e);
  return (uint16_t)(lo | hi << 8);
}
__device__ __forceinline__ uint32_t join_notes(uint4 v) {
  const uint32_t w = __vmaxu4(__vmaxu4(v.x, v.y), __vmaxu4(v.z, v.w));
  return __vmaxu4(w, w >> 16) & 0xffffu;
}
constexpr uint32_t NOTE_ORDINARY = (255 - (127 - 63)) | (127 + 62) << 8;  // within 2^-63 .. 2^63
// Powers of two that hold the noted scales between them; 0 and 0 without any.
__device__ __forceinline__ float note_least(uint32_t n) {
  return (n >> 8) ? __uint_as_float((255u - (n & 255u)) << 23) : 0.f;
}
__device__ __forceinline__ float note_most(uint32_t n) {
  return (n >> 8) ? __uint_as_float(((n >> 8) + 1u) << 23) : 0.f;
}

}  // namespace aqtb200
