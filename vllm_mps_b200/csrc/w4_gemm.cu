// Products with 4-bit weights and group scales, for a few activation rows:
//   Y[m][n] = sum_g scale[n][g] * sum_{k in g} X[m][k] * (code[n][k] - zero[n][g])
// optionally with the gated-MLP epilogue on a fused [gate; up] weight,
//   Y[m][i] = silu(gate[m][i]) * up[m][i].
//
// One warp per output feature: its lanes walk the row 8 codes at a time, each
// group's sum of code products and of activations is kept apart in fp32 and
// scaled once.
#include "vmps_abi_internal.h"
#include "vmps_common.cuh"

namespace vmps {
namespace {

constexpr int kW4MaxRows = 32;
constexpr int kW4Warps = 8;

struct W4Params {
  void* out;
  int64_t out_stride;
  const void* x;
  int64_t x_stride;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;  // NULL: 8
  int M, N, K, group, silu;
};

template <typename T>
__device__ float w4_dot(const W4Params& p, int m, int row, int lane) {
  const T* x = static_cast<const T*>(p.x) + m * p.x_stride;
  const int ng = p.K / p.group;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p.codes + static_cast<int64_t>(row) * (p.K / 2));
  const T* sc = static_cast<const T*>(p.scales) + static_cast<int64_t>(row) * ng;
  float acc = 0.f;
  for (int k = lane * 8; k < p.K; k += 256) {
    const uint32_t v = w[k / 8];
    const int g = k / p.group;
    const float z = p.zeros ? static_cast<float>(p.zeros[static_cast<int64_t>(row) * ng + g]) : 8.f;
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      part += Elt<T>::to_f(x[k + j]) * (static_cast<float>((v >> (4 * j)) & 15u) - z);
    }
    acc += part * Elt<T>::to_f(sc[g]);
  }
  for (int sh = 16; sh; sh >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, sh);
  return acc;
}

template <typename T>
__global__ void __launch_bounds__(32 * kW4Warps) w4_kernel(const W4Params p) {
  const int row = blockIdx.x * kW4Warps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.N) return;
  T* out = static_cast<T*>(p.out);
  for (int m = 0; m < p.M; ++m) {
    float y = w4_dot<T>(p, m, row, lane);
    if (p.silu) {
      const float u = w4_dot<T>(p, m, row + p.N, lane);
      y = y / (1.f + expf(-y)) * u;
    }
    if (lane == 0) out[m * p.out_stride + row] = Elt<T>::from_f(y);
  }
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" int vmps_w4_gemm_supported(int M, int N, int K, int group_size) {
  if (M < 0 || M > kW4MaxRows || N <= 0 || K <= 0) return 0;
  if (group_size != 32 && group_size != 64 && group_size != 128) return 0;
  return K % group_size == 0 ? 1 : 0;
}

extern "C" int vmps_w4_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                            const void* codes, const void* scales, const void* zeros, int M, int N,
                            int K, int group_size, int silu_mul, int dtype, void* stream) {
  const char* what = "w4_gemm";
  clear_error();
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (!vmps_w4_gemm_supported(M, N, K, group_size)) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: M=%d N=%d K=%d group=%d (M <= %d, group 32, 64 or 128, K a multiple of it)",
                what, M, N, K, group_size, kW4MaxRows);
  }
  if (M == 0) return VMPS_OK;
  if (!out || !x || !codes || !scales) return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  if (x_row_stride < K || out_row_stride < N) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: row stride smaller than a row", what);
  }
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || (zeros && !aligned16(zeros)) ||
      (x_row_stride % 8) || (reinterpret_cast<uintptr_t>(out) & 1)) {
    return fail(VMPS_ERR_ALIGNMENT,
                "%s: x, codes, scales and zeros must be 16-byte aligned, x rows a multiple of 8 "
                "elements apart, out 2-byte aligned",
                what);
  }
  W4Params p;
  p.out = out;
  p.out_stride = out_row_stride;
  p.x = x;
  p.x_stride = x_row_stride;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.M = M;
  p.N = N;
  p.K = K;
  p.group = group_size;
  p.silu = silu_mul ? 1 : 0;
  const int grid = (N + kW4Warps - 1) / kW4Warps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) w4_kernel<__half><<<grid, 32 * kW4Warps, 0, s>>>(p);
  else w4_kernel<__nv_bfloat16><<<grid, 32 * kW4Warps, 0, s>>>(p);
  return check_launch(what);
}
