// The 8-bit paged cache: its two code formats and their layout.
//
//   codes  [num_blocks][2][16][n_kv][D]  int8 or e4m3 (dim 1: 0 = K, 1 = V)
//   scales [num_blocks][n_kv][2][16]     fp32
//
// A stored value is code * scale.  A token's D values of one head share a
// scale: their largest magnitude over the largest code (127, 448).  The scales
// of a page lie together by head, K's 16 and then V's, so that a head group's
// are one contiguous piece.
#pragma once

#include <cuda_fp8.h>

#include "vmps_common.cuh"

namespace vmps {

constexpr int kCachePage = 16;

// Rows whose largest magnitude is below this are stored as zeros (127 over a
// smaller one would leave fp32's range).
constexpr float kCache8Tiny = 7.888609052210118e-31f;  // 2^-100

struct Int8Code {
  static constexpr float kTop = 127.f;
  // Nearest integer, ties to even; |y| <= 127 (1 + 2^-22).
  static __device__ __forceinline__ uint32_t code(float y) {
    return static_cast<uint32_t>(__float2int_rn(y)) & 0xffu;
  }
  // Four codes at once, the first in the lowest byte.
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
  }
  static __device__ __forceinline__ void unpack4(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xffu));
    }
  }
};

struct E4m3Code {
  static constexpr float kTop = 448.f;
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  static __device__ __forceinline__ void unpack4(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((w >> (16 * i)) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

}  // namespace vmps
