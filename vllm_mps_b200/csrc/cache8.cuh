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

#include <utility>

#include "vmps_common.cuh"

namespace vmps {

constexpr int kCachePage = 16;

// Rows whose largest magnitude is below this are stored as zeros (127 over a
// smaller one would leave fp32's range).
constexpr float kCache8Tiny = 7.888609052210118e-31f;  // 2^-100

// Two fp32 values in one 64-bit register: Blackwell multiplies and adds both at once.
using f2 = unsigned long long;

__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(f2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The codes' quotients x * top / a of a row whose largest magnitude is a (2^-100 to 2^128).
// 16-bit values lie on ties often (x = a / 2 is 63.5 steps), and the product with a rounded
// reciprocal puts those on either side; so the quotient is corrected by its remainder, which
// the fused multiply-add gives exactly (Markstein's division): 16-bit values go to the code
// that the exact quotient is nearest to.  a's power of two is taken off both beforehand.
struct Quotient {
  f2 up, down, inv;
  __device__ __forceinline__ Quotient(float a, float top) {
    const uint32_t bits = __float_as_uint(a);
    const float t = 0.5f * top * __uint_as_float((255u << 23) - (bits & 0x7f800000u));
    const float m = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u), r = __frcp_rn(m);
    up = pair(t, t);
    down = pair(-m, -m);
    inv = pair(r, r);
  }
  __device__ __forceinline__ f2 operator()(f2 x) const {
    const f2 n = mul2(x, up), y = mul2(n, inv);
    return fma2(fma2(y, down, n), inv, y);
  }
};

struct Int8Code {
  static constexpr float kTop = 127.f;
  // Codes of four quotients, the first in the lowest byte: the nearest integer, ties to even,
  // is the low byte of 1.5 * 2^23 plus it (at most 127 (1 + 2^-22)).
  static __device__ __forceinline__ uint32_t pack4(f2 x, f2 y) {
    constexpr float kBase = 12582912.f;
    const float2 lo = split(add2(x, pair(kBase, kBase))), hi = split(add2(y, pair(kBase, kBase)));
    const uint32_t ab = __byte_perm(__float_as_uint(lo.x), __float_as_uint(lo.y), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(hi.x), __float_as_uint(hi.y), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
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
  static __device__ __forceinline__ uint32_t pack4(f2 x, f2 y) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(split(x), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(split(y), __NV_SATFINITE, __NV_E4M3);
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

// The 8-bit cache's kernels are links of a chain of kernels launched with programmatic
// dependent launch: each waits for what is before it on the stream before it reads
// anything, and only then lets the next one start.
__device__ __forceinline__ void chain_link() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// `early`: whether the launch may start before what is ahead of it has ended.
template <typename... KArgs, typename... Args>
cudaError_t launch_link(void (*kernel)(KArgs...), bool early, dim3 grid, dim3 block, size_t smem,
                        cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace vmps
