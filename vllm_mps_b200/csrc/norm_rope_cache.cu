// Kernel 9: norms of queries and keys per head, the position rotation and the
// cache write in one pass, into a 16-bit pool or the 8-bit cache.
//
//   y = x * w / sqrt(mean(x^2) + eps)                    (weights optional)
//   z[j]       = y[j] cos a_j - y[j + D/2] sin a_j
//   z[j + D/2] = y[j + D/2] cos a_j + y[j] sin a_j,      a_j = position * inv_freq[j]
//
// for q and k; v is cached as it is.  Everything between the input and the
// result is fp32 (the angle, whose quarter turns are taken off, in 64 bits) and
// the result is rounded once: to the 16-bit type, or to a code.
//
// What bounds it: the bytes of q, k and v in and out; 8192 rows of 32/8 heads x
// 128 into the int8 cache take 35.4 us (5.2 TB/s; the instructions keep 67 % of the
// issue slots), one row 2.1 us.  What hides the loads is the number of warps: with
// 72 registers and 28 warps an SM 34.7 us (before the codes' quotients were
// corrected), with 80 and 24 39, with 64 and 32, where a few values are spilled, 36.9.
#include "cache8.cuh"
#include "rows_overlap.h"
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
  int parts, steps;  // warps that share a row, steps of each
  int64_t num_rows, num_slots;
  int* err;
};

// Cosine and sine of position * inv_freq.  The product is exact to 2^-53; its
// quarter turns are taken off in 64 bits (pi / 2 in two parts; adding 1.5 * 2^52
// leaves their number in the sum's low bits), so that far positions keep the
// accuracy of near ones.  What is left is at most pi / 4, where Taylor's sums up
// to r^9 and r^10 are within 2^-28 of the functions.
__device__ __forceinline__ void rotation(int pos, float inv_freq, float* cs, float* sn) {
  const double a = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double t = fma(a, 0.6366197723675814, 6755399441055744.0);
  const int quarter = __double2loint(t);
  const double n = t - 6755399441055744.0;
  const float r = static_cast<float>(fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a)));
  const float z = r * r;
  float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = fmaf(z, s, 1.f / 120.f);
  s = fmaf(z, s, -1.f / 6.f);
  s = fmaf(z * r, s, r);
  float c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  c = fmaf(z, c, -1.f / 720.f);
  c = fmaf(z, c, 1.f / 24.f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  const float x = (quarter & 1) ? s : c, y = (quarter & 1) ? c : s;
  *cs = ((quarter + 1) & 2) ? -x : x;
  *sn = (quarter & 2) ? -y : y;
}

// NaN if one of them is (0x7fffffff, above every number's bits).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, f2 (&x)[4]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      x[i] = pair(f.x, f.y);
    } else {
      x[i] = pair(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u));
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const f2 (&x)[4]) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = split(x[i]);
    v[i] = Elt<T>::pack(f.x, f.y);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
}

constexpr int kStoreWarps = 4;     // of a block
constexpr int kStoreResident = 7;  // blocks of an SM

// D / 16 lanes share a head: lane c holds elements 8c.. of each half, so that a
// rotated pair is in one lane; a warp takes 512 / D heads a step.  A warp works
// by itself on up to p.steps steps of one row, the next one's values on their way.
// It works the row's angles out once, two a lane (one at head size 64), and hands
// them round.
template <typename T, int D, typename Code>
__global__ void __launch_bounds__(32 * kStoreWarps, kStoreResident)
norm_rope_cache_kernel(const StoreParams p) {
  constexpr int kHalf = D / 2;
  constexpr int kLanes = D / 16;
  constexpr int kHeads = 32 / kLanes;  // of a step
  constexpr int kAngles = kHalf / 32;  // of a lane
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kStoreWarps + threadIdx.x / 32;
  chain_link();
  const int64_t i = item / p.parts;
  if (i >= p.num_rows) return;
  const int heads = p.n_q + 2 * p.n_kv;
  const int c = lane % kLanes;
  const int first = static_cast<int>(item % p.parts) * p.steps * kHeads;
  const int end = min(first + p.steps * kHeads, heads);

  // A lane without a head works on the last one and stores nothing: whole warps take part
  // in the shuffles.
  const T* const q = static_cast<const T*>(p.q) + i * p.q_stride + c * 8;
  const T* const k = static_cast<const T*>(p.k) + i * p.k_stride + c * 8;
  const T* const v = static_cast<const T*>(p.v) + i * p.v_stride + c * 8;
  auto load = [&](int h0, uint4& lo, uint4& hi) {
    int h = min(h0 + lane / kLanes, heads - 1);
    const T* src = q;
    if (h >= p.n_q) {
      h -= p.n_q;
      src = k;
      if (h >= p.n_kv) {
        h -= p.n_kv;
        src = v;
      }
    }
    src += static_cast<int64_t>(h) * D;
    lo = *reinterpret_cast<const uint4*>(src);
    hi = *reinterpret_cast<const uint4*>(src + kHalf);
  };
  uint4 lo4, hi4;
  load(first, lo4, hi4);
  const bool rotate = p.inv_freq != nullptr;
  const int pos = rotate ? p.positions[i] : 0;
  const int64_t slot = p.slot_mapping[i];
  if (pos < 0) {
    if (lane == 0) set_error(p.err, kDevErrPositionRange);
    return;
  }
  if (slot >= p.num_slots && lane == 0) set_error(p.err, kDevErrSlotRange);
  const bool write = slot >= 0 && slot < p.num_slots;
  const int64_t blk = write ? slot / kCachePage : 0;
  const int64_t off = write ? slot % kCachePage : 0;
  f2 cs[4], sn[4];
  if (rotate) {
    float mc[kAngles], ms[kAngles];
#pragma unroll
    for (int a = 0; a < kAngles; ++a) {
      rotation(pos, p.inv_freq[lane * kAngles + a], &mc[a], &ms[a]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int f0 = (8 * c + 2 * e) / kAngles, f1 = (8 * c + 2 * e + 1) / kAngles;
      cs[e] = pair(__shfl_sync(0xffffffffu, mc[0], f0), __shfl_sync(0xffffffffu, mc[kAngles - 1], f1));
      sn[e] = pair(__shfl_sync(0xffffffffu, ms[0], f0), __shfl_sync(0xffffffffu, ms[kAngles - 1], f1));
    }
  }
#pragma unroll 1
  for (int h0 = first; h0 < end; h0 += kHeads) {
    const bool live = h0 + lane / kLanes < end;
    const int h = min(h0 + lane / kLanes, heads - 1);
    const bool is_q = h < p.n_q;
    const bool is_v = h >= p.n_q + p.n_kv;
    const int hk = is_q ? h : is_v ? h - p.n_q - p.n_kv : h - p.n_q;
    f2 lo[4], hi[4];
    unpack8<T>(lo4, lo);
    unpack8<T>(hi4, hi);
    if (h0 + kHeads < end) load(h0 + kHeads, lo4, hi4);
    // (A step of one kind skips what only others need.)
    if ((p.q_weight && h0 < p.n_q) ||
        (p.k_weight && h0 < p.n_q + p.n_kv && h0 + kHeads > p.n_q)) {
      f2 sums = pair(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) sums = fma2(hi[e], hi[e], fma2(lo[e], lo[e], sums));
      const float2 two = split(sums);
      float sum = two.x + two.y;
#pragma unroll
      for (int sh = 1; sh < kLanes; sh <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
      const T* weight = static_cast<const T*>(is_q ? p.q_weight : is_v ? nullptr : p.k_weight);
      if (weight) {
        const float scale = rsqrtf(sum * (1.f / D) + p.eps);
        const f2 scale2 = pair(scale, scale);
        f2 wl[4], wh[4];
        unpack8<T>(*reinterpret_cast<const uint4*>(weight + c * 8), wl);
        unpack8<T>(*reinterpret_cast<const uint4*>(weight + kHalf + c * 8), wh);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = mul2(lo[e], mul2(scale2, wl[e]));
          hi[e] = mul2(hi[e], mul2(scale2, wh[e]));
        }
      }
    }
    if (rotate && !is_v) {
      const f2 minus = pair(-1.f, -1.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f2 a = fma2(lo[e], cs[e], mul2(mul2(hi[e], sn[e]), minus));
        hi[e] = fma2(hi[e], cs[e], mul2(lo[e], sn[e]));
        lo[e] = a;
      }
    }
    if (is_q) {
      if (live) {
        T* dst = static_cast<T*>(p.q_out) + i * p.q_out_stride + static_cast<int64_t>(hk) * D + c * 8;
        store8(dst, lo);
        store8(dst + kHalf, hi);
      }
    }
    if (h0 + kHeads <= p.n_q) continue;
    const bool mine = live && !is_q && write;
    if constexpr (!std::is_void<Code>::value) {
      // The largest magnitude, as bits: infinities and NaN are above every number.
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a = split(lo[e]), b = split(hi[e]);
        most = max3(most, fabsf(a.x), fabsf(a.y));
        most = max3(most, fabsf(b.x), fabsf(b.y));
      }
      uint32_t top = __float_as_uint(most);
#pragma unroll
      for (int sh = 1; sh < kLanes; sh <<= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, sh));
      }
      if (mine) {
        const float a = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;
        const bool some = finite && a >= kCache8Tiny;
        uint2 wl = make_uint2(0u, 0u), wh = make_uint2(0u, 0u);
        if (some) {
          const Quotient over(a, Code::kTop);
          wl = make_uint2(Code::pack4(over(lo[0]), over(lo[1])), Code::pack4(over(lo[2]), over(lo[3])));
          wh = make_uint2(Code::pack4(over(hi[0]), over(hi[1])), Code::pack4(over(hi[2]), over(hi[3])));
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
    } else if (mine) {
      T* dst = static_cast<T*>(p.cache) +
               (((blk * 2 + (is_v ? 1 : 0)) * kCachePage + off) * p.n_kv + hk) * D + c * 8;
      store8(dst, lo);
      store8(dst + kHalf, hi);
    }
  }
}

// Steps of a warp, at most (8192 rows of 32/8 heads, head size 128, 12 steps: 34.7 us with
// 12, 36.5 with 6; rows of 18 and 30 steps gain nothing from more).
constexpr int kSteps = 12;

template <typename T, int D, typename Code>
int launch_store(StoreParams p, cudaStream_t s) {
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  // Steps of a row, and the warps that share them: the fewest steps one after the other over
  // all waves of warps, of which each costs two steps more (400 rows of 32/8 heads x 128 with
  // 3 steps a warp 3.8 us, 5.4 with 6 (64 registers); 1000 rows of 40/40 heads 13.0 and 15.9).
  const int all = ((p.n_q + 2 * p.n_kv) * (D / 16) + 31) / 32;
  int64_t best = INT64_MAX;
  for (int most = 1; most <= kSteps; ++most) {
    const int parts = (all + most - 1) / most, steps = (all + parts - 1) / parts;
    const int64_t warps = static_cast<int64_t>(kStoreResident) * kStoreWarps * sms;
    const int64_t waves = (p.num_rows * parts + warps - 1) / warps;
    if (waves * (steps + 2) <= best) {
      best = waves * (steps + 2);
      p.parts = parts;
      p.steps = steps;
    }
  }
  const int64_t items = p.num_rows * p.parts;
  const int64_t grid = (items + kStoreWarps - 1) / kStoreWarps;
  if (grid > 0x7fffffff) return fail(VMPS_ERR_UNSUPPORTED, "norm_rope_and_cache: too many rows");
  // An early start saves small calls 0.4 us; the blocks of larger grids are then spread
  // unevenly over the SMs that the launch before still holds (2000 rows of 40 heads x 64:
  // 6.1 -> 7.7 us).
  const cudaError_t e = launch_link(norm_rope_cache_kernel<T, D, Code>, grid <= sms,
                                    dim3((unsigned)grid), dim3(32 * kStoreWarps), 0, s, p);
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "norm_rope_and_cache: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
}

template <typename T, int D>
int launch_store(const StoreParams& p, int format, cudaStream_t s) {
  switch (format) {
    case VMPS_CACHE_16BIT: return launch_store<T, D, void>(p, s);
    case VMPS_CACHE_INT8: return launch_store<T, D, Int8Code>(p, s);
    default: return launch_store<T, D, E4m3Code>(p, s);
  }
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
  // Rows are read and written by several warps in no order.
  const bool in_place = q_out == q && (num_rows == 1 || q_out_row_stride == q_row_stride);
  if ((!in_place && rows_overlap(q_out, q_out_row_stride * 2, q_row * 2, q, q_row_stride * 2,
                                 q_row * 2, num_rows)) ||
      rows_overlap(q_out, q_out_row_stride * 2, q_row * 2, k, k_row_stride * 2, kv_row * 2, num_rows) ||
      rows_overlap(q_out, q_out_row_stride * 2, q_row * 2, v, v_row_stride * 2, kv_row * 2, num_rows)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: q_out overlaps q (but is not q), k or v", what);
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
  p.num_rows = num_rows;
  p.num_slots = static_cast<int64_t>(num_blocks) * kCachePage;
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_store<__half, 64>(p, cache_format, s)
                          : launch_store<__half, 128>(p, cache_format, s);
  }
  return head_dim == 64 ? launch_store<__nv_bfloat16, 64>(p, cache_format, s)
                        : launch_store<__nv_bfloat16, 128>(p, cache_format, s);
}

extern "C" int vmps_norm_rope_and_cache_args(const vmps_norm_rope_args* a, void* stream) {
  if (!a) return vmps::fail(VMPS_ERR_INVALID_ARG, "norm_rope_and_cache: NULL arguments");
  return vmps_norm_rope_and_cache(a->q_out, a->q_out_row_stride, a->q, a->q_row_stride, a->k,
                                  a->k_row_stride, a->v, a->v_row_stride, a->q_weight, a->k_weight,
                                  a->eps, a->positions, a->slot_mapping, a->inv_freq, a->cache,
                                  a->scales, a->num_rows, a->n_q, a->n_kv, a->head_dim,
                                  a->block_size, a->num_blocks, a->cache_format, a->dtype, stream);
}
