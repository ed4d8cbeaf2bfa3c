// Kernel 9: norms of queries and keys per head, the position rotation and the
// cache write in one pass, into a 16-bit pool or the 8-bit cache.
//
//   y = x * w / sqrt(mean(x^2) + eps)                    (weights optional)
//   z[j]       = y[j] cos a_j - y[j + D/2] sin a_j
//   z[j + D/2] = y[j + D/2] cos a_j + y[j] sin a_j,      a_j = position * inv_freq[j]
//
// for q and k; v is cached as it is.  Everything between the input and the
// result is fp32 (the angle, whose whole turns are taken off, in 64 bits) and
// the result is rounded once: to the 16-bit type, or to a code.
#include "cache8.cuh"
#include "vmps_abi_internal.h"

namespace vmps {
namespace {

struct StoreParams {
  void* q_out;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_out_stride, q_stride, k_stride, v_stride;  // elements between rows
  const void* q_weight;
  const void* k_weight;
  float eps;
  const int32_t* positions;
  const int32_t* slot_mapping;
  const float* inv_freq;
  void* cache;
  float* scales;
  int n_q, n_kv;
  int64_t num_slots;
  int* err;
};

// Cosine and sine of position * inv_freq.  The product is exact to 2^-53; its
// whole turns are taken off in 64 bits (2 pi in two parts), so that far
// positions keep the accuracy of near ones, and the rest is at most pi.
__device__ __forceinline__ void rotation(int pos, float inv_freq, float* cs, float* sn) {
  const double a = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double n = rint(a * 0.15915494309189535);
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
  sincosf(static_cast<float>(r), sn, cs);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Elt<T>::to_f(e[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(Elt<T>::pack(x[0], x[1]), Elt<T>::pack(x[2], x[3]), Elt<T>::pack(x[4], x[5]),
                 Elt<T>::pack(x[6], x[7]));
}

// D / 16 lanes share a head: lane c holds elements 8c.. of each half, so that a
// rotated pair is in one lane.
template <typename T, int D, typename Code>
__global__ void __launch_bounds__(512) norm_rope_cache_kernel(const StoreParams p) {
  constexpr int kHalf = D / 2;
  constexpr int kLanes = D / 16;
  __shared__ float s_cos[kHalf];
  __shared__ float s_sin[kHalf];

  const int64_t i = blockIdx.x;
  const bool rotate = p.inv_freq != nullptr;
  const int pos = rotate ? p.positions[i] : 0;
  if (pos < 0) {
    if (threadIdx.x == 0) set_error(p.err, kDevErrPositionRange);
    return;
  }
  if (rotate) {
    for (int j = threadIdx.x; j < kHalf; j += blockDim.x) {
      rotation(pos, p.inv_freq[j], &s_cos[j], &s_sin[j]);
    }
    __syncthreads();
  }
  const int64_t slot = p.slot_mapping[i];
  const bool write = slot >= 0 && slot < p.num_slots;
  if (slot >= p.num_slots && threadIdx.x == 0) set_error(p.err, kDevErrSlotRange);
  const int64_t blk = write ? slot / kCachePage : 0;
  const int64_t off = write ? slot % kCachePage : 0;

  const int c = threadIdx.x % kLanes;
  const int heads = p.n_q + 2 * p.n_kv;
  // Whole warps take part in the shuffles; a lane group without a head works on
  // the last one and stores nothing.
  const int per_pass = blockDim.x / kLanes;
  for (int h0 = 0; h0 < heads; h0 += per_pass) {
    const int hh = h0 + static_cast<int>(threadIdx.x) / kLanes;
    const bool live = hh < heads;
    const int h = live ? hh : heads - 1;
    const bool is_q = h < p.n_q;
    const bool is_v = h >= p.n_q + p.n_kv;
    const int hk = is_q ? h : is_v ? h - p.n_q - p.n_kv : h - p.n_q;
    const T* src = is_q   ? static_cast<const T*>(p.q) + i * p.q_stride
                   : is_v ? static_cast<const T*>(p.v) + i * p.v_stride
                          : static_cast<const T*>(p.k) + i * p.k_stride;
    src += static_cast<int64_t>(hk) * D + c * 8;
    float lo[8], hi[8];
    load8(src, lo);
    load8(src + kHalf, hi);
    const T* weight = static_cast<const T*>(is_q ? p.q_weight : is_v ? nullptr : p.k_weight);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
    for (int sh = 1; sh < kLanes; sh <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
    if (weight) {
      const float r = rsqrtf(sum * (1.f / D) + p.eps);
      float wl[8], wh[8];
      load8(weight + c * 8, wl);
      load8(weight + kHalf + c * 8, wh);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] *= r * wl[e];
        hi[e] *= r * wh[e];
      }
    }
    if (rotate && !is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float cs = s_cos[c * 8 + e], sn = s_sin[c * 8 + e];
        const float a = lo[e] * cs - hi[e] * sn;
        hi[e] = hi[e] * cs + lo[e] * sn;
        lo[e] = a;
      }
    }
    if constexpr (!std::is_void<Code>::value) {
      // The largest magnitude, as bits: infinities and NaN are above every number.
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = max(top, __float_as_uint(lo[e]) & 0x7fffffffu);
        top = max(top, __float_as_uint(hi[e]) & 0x7fffffffu);
      }
#pragma unroll
      for (int sh = 1; sh < kLanes; sh <<= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, sh));
      }
      if (live && !is_q && write) {
        const float a = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;
        const bool some = finite && a >= kCache8Tiny;
        const float inv = some ? Code::kTop / a : 0.f;
        uint2 wl = make_uint2(0u, 0u), wh = make_uint2(0u, 0u);
        if (some) {
          wl = make_uint2(Code::pack4(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv),
                          Code::pack4(lo[4] * inv, lo[5] * inv, lo[6] * inv, lo[7] * inv));
          wh = make_uint2(Code::pack4(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv),
                          Code::pack4(hi[4] * inv, hi[5] * inv, hi[6] * inv, hi[7] * inv));
        }
        uint8_t* dst = static_cast<uint8_t*>(p.cache) +
                       (((blk * 2 + (is_v ? 1 : 0)) * kCachePage + off) * p.n_kv + hk) * D + c * 8;
        *reinterpret_cast<uint2*>(dst) = wl;
        *reinterpret_cast<uint2*>(dst + kHalf) = wh;
        if (c == 0) {
          p.scales[((blk * p.n_kv + hk) * 2 + (is_v ? 1 : 0)) * kCachePage + off] =
              some ? a / Code::kTop : finite ? 0.f : __uint_as_float(0x7fc00000u);
        }
      }
    } else if (live && !is_q && write) {
      T* dst = static_cast<T*>(p.cache) +
               (((blk * 2 + (is_v ? 1 : 0)) * kCachePage + off) * p.n_kv + hk) * D + c * 8;
      store8(dst, lo);
      store8(dst + kHalf, hi);
    }
    if (live && is_q) {
      T* dst = static_cast<T*>(p.q_out) + i * p.q_out_stride + static_cast<int64_t>(hk) * D + c * 8;
      store8(dst, lo);
      store8(dst + kHalf, hi);
    }
  }
}

template <typename T, int D>
int launch_store(const StoreParams& p, int rows, int format, cudaStream_t s) {
  const int threads = min(512, ((p.n_q + 2 * p.n_kv) * (D / 16) + 31) / 32 * 32);
  switch (format) {
    case VMPS_CACHE_16BIT:
      norm_rope_cache_kernel<T, D, void><<<rows, threads, 0, s>>>(p);
      break;
    case VMPS_CACHE_INT8:
      norm_rope_cache_kernel<T, D, Int8Code><<<rows, threads, 0, s>>>(p);
      break;
    default:
      norm_rope_cache_kernel<T, D, E4m3Code><<<rows, threads, 0, s>>>(p);
      break;
  }
  return check_launch("norm_rope_and_cache");
}

}  // namespace
}  // namespace vmps

extern "C" int vmps_norm_rope_and_cache(
    void* q_out, int64_t q_out_row_stride, const void* q, int64_t q_row_stride, const void* k,
    int64_t k_row_stride, const void* v, int64_t v_row_stride, const void* q_weight,
    const void* k_weight, float eps, const int32_t* positions, const int32_t* slot_mapping,
    const float* inv_freq, void* cache, float* scales, int num_rows, int n_q, int n_kv,
    int head_dim, int block_size, int num_blocks, int cache_format, int dtype, void* stream) {
  using namespace vmps;
  clear_error();
  const char* what = "norm_rope_and_cache";
  if (num_rows < 0 || n_q < 0 || n_kv <= 0 || num_blocks <= 0 || n_q > (1 << 16) ||
      n_kv > (1 << 16)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: bad sizes (num_rows=%d n_q=%d n_kv=%d num_blocks=%d)",
                what, num_rows, n_q, n_kv, num_blocks);
  }
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (cache_format < VMPS_CACHE_16BIT || cache_format > VMPS_CACHE_E4M3) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: cache_format %d", what, cache_format);
  }
  if (head_dim != 64 && head_dim != 128) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  }
  if (block_size != kCachePage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  if (num_rows == 0) return VMPS_OK;
  if ((n_q > 0 && (!q || !q_out)) || !k || !v || !cache || !slot_mapping ||
      (inv_freq && !positions) || (cache_format != VMPS_CACHE_16BIT && !scales)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  }
  if ((n_q > 0 && (!aligned16(q) || !aligned16(q_out) || (q_row_stride % 8) ||
                   (q_out_row_stride % 8))) ||
      !aligned16(k) || !aligned16(v) || !aligned16(cache) || (k_row_stride % 8) ||
      (v_row_stride % 8) || !aligned16(q_weight) || !aligned16(k_weight)) {
    return fail(VMPS_ERR_ALIGNMENT,
                "%s: pointers must be 16-byte aligned and row strides multiples of 8 elements",
                what);
  }
  if (reinterpret_cast<uintptr_t>(scales) & 3) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: scales must be 4-byte aligned", what);
  }
  const int64_t q_row = static_cast<int64_t>(n_q) * head_dim;
  const int64_t kv_row = static_cast<int64_t>(n_kv) * head_dim;
  if (num_rows > 1 && (q_row_stride < q_row || q_out_row_stride < q_row || k_row_stride < kv_row ||
                       v_row_stride < kv_row)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: row stride smaller than a row", what);
  }
  if (!(eps >= 0.f)) return fail(VMPS_ERR_INVALID_ARG, "%s: eps %g", what, (double)eps);
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  StoreParams p;
  p.q_out = q_out;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out_stride = q_out_row_stride;
  p.q_stride = q_row_stride;
  p.k_stride = k_row_stride;
  p.v_stride = v_row_stride;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.eps = eps;
  p.positions = positions;
  p.slot_mapping = slot_mapping;
  p.inv_freq = inv_freq;
  p.cache = cache;
  p.scales = scales;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.num_slots = static_cast<int64_t>(num_blocks) * kCachePage;
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_store<__half, 64>(p, num_rows, cache_format, s)
                          : launch_store<__half, 128>(p, num_rows, cache_format, s);
  }
  return head_dim == 64 ? launch_store<__nv_bfloat16, 64>(p, num_rows, cache_format, s)
                        : launch_store<__nv_bfloat16, 128>(p, num_rows, cache_format, s);
}
