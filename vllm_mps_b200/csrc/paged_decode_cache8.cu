// Kernel 11: decode attention over the 8-bit paged cache, one query token per
// sequence.
//
//   out[i][h] = softmax_t(scale * q[i][h] . K[t]) . V[t],  K, V = code * scale
#include "cache8.cuh"
#include "vmps_abi_internal.h"

namespace vmps {
namespace {

constexpr int kMaxSeqs8 = 4096;
constexpr int kMaxKvHeads8 = 64;
constexpr int kMaxGroup8 = 16;

struct Decode8Params {
  void* out;
  const void* q;
  int64_t q_stride;
  const uint8_t* codes;
  const float* scales;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  int max_blocks, n_kv, G, num_blocks;
  float scale_log2;
  int* err;
};

// One warp takes every fourth token; a lane owns D / 32 elements.
template <typename T, int D, typename Code>
__global__ void __launch_bounds__(128) decode8_kernel(const Decode8Params p) {
  constexpr int kE = D / 32;
  __shared__ float s_m[4][kMaxGroup8], s_l[4][kMaxGroup8], s_o[4][kMaxGroup8][D];
  const int kvh = blockIdx.x, s = blockIdx.y;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int len = max(p.seq_lens[s], 0);
  if (len > p.max_blocks * kCachePage) {
    if (threadIdx.x == 0) set_error(p.err, kDevErrSeqLen);
    len = p.max_blocks * kCachePage;
  }
  const T* q = static_cast<const T*>(p.q) + s * p.q_stride + static_cast<int64_t>(kvh) * p.G * D;
  float qf[kMaxGroup8][kE], o[kMaxGroup8][kE], m[kMaxGroup8], l[kMaxGroup8];
  for (int g = 0; g < kMaxGroup8; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
    for (int e = 0; e < kE; ++e) {
      qf[g][e] = g < p.G ? Elt<T>::to_f(q[g * D + lane * kE + e]) : 0.f;
      o[g][e] = 0.f;
    }
  }
  for (int t = warp; t < len; t += 4) {
    const int blk = p.block_tables[static_cast<int64_t>(s) * p.max_blocks + t / kCachePage];
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) set_error(p.err, kDevErrBlockRange);
      continue;
    }
    const int64_t at = (static_cast<int64_t>(blk) * 2 * kCachePage + t % kCachePage) * p.n_kv + kvh;
    const float* sc = p.scales + (static_cast<int64_t>(blk) * p.n_kv + kvh) * 2 * kCachePage + t % kCachePage;
    float k[kE], v[kE];
    for (int e = 0; e < kE; ++e) {
      float x[4];
      Code::unpack4(p.codes[at * D + lane * kE + e], x);
      k[e] = x[0] * sc[0];
      Code::unpack4(p.codes[(at + static_cast<int64_t>(kCachePage) * p.n_kv) * D + lane * kE + e], x);
      v[e] = x[0] * sc[kCachePage];
    }
    for (int g = 0; g < kMaxGroup8; ++g) {
      if (g >= p.G) break;
      float x = 0.f;
      for (int e = 0; e < kE; ++e) x += qf[g][e] * k[e];
      for (int sh = 16; sh; sh >>= 1) x += __shfl_xor_sync(0xffffffffu, x, sh);
      x *= p.scale_log2;
      const float mn = fmaxf(m[g], x);
      const float al = mn == m[g] ? 1.f : exp2f(m[g] - mn), w = exp2f(x - mn);
      m[g] = mn;
      l[g] = l[g] * al + w;
      for (int e = 0; e < kE; ++e) o[g][e] = o[g][e] * al + w * v[e];
    }
  }
  for (int g = 0; g < p.G; ++g) {
    s_m[warp][g] = m[g];
    s_l[warp][g] = l[g];
    for (int e = 0; e < kE; ++e) s_o[warp][g][lane * kE + e] = o[g][e];
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(s) * p.n_kv + kvh) * p.G * D;
  for (int i = threadIdx.x; i < p.G * D; i += blockDim.x) {
    const int g = i / D, d = i % D;
    float mm = -INFINITY, ll = 0.f, x = 0.f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w][g]);
    for (int w = 0; w < 4; ++w) {
      if (s_l[w][g] == 0.f) continue;  // no token
      const float f = exp2f(s_m[w][g] - mm);
      ll += s_l[w][g] * f;
      x += s_o[w][g][d] * f;
    }
    out[i] = Elt<T>::from_f(len > 0 ? x / ll : 0.f);
  }
}

template <typename T, int D>
int launch_decode8(const Decode8Params& p, int num_seqs, int format, cudaStream_t s) {
  const dim3 grid(p.n_kv, num_seqs);
  if (format == VMPS_CACHE_INT8) {
    decode8_kernel<T, D, Int8Code><<<grid, 128, 0, s>>>(p);
  } else {
    decode8_kernel<T, D, E4m3Code><<<grid, 128, 0, s>>>(p);
  }
  return check_launch("paged_decode_attention_cache8");
}

}  // namespace
}  // namespace vmps

extern "C" size_t vmps_paged_decode_cache8_workspace_bytes(int num_seqs, int n_q, int n_kv,
                                                           int head_dim) {
  using namespace vmps;
  if (num_seqs < 0 || num_seqs > kMaxSeqs8 || n_kv <= 0 || n_kv > kMaxKvHeads8 || n_q <= 0 ||
      n_q % n_kv || n_q / n_kv > kMaxGroup8 || (head_dim != 64 && head_dim != 128)) {
    return 0;
  }
  return 256;
}

extern "C" int vmps_paged_decode_attention_cache8(
    void* out, const void* q, int64_t q_row_stride, const void* codes, const float* scales,
    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* seq_lens, int num_seqs,
    int n_q, int n_kv, int head_dim, int block_size, int num_blocks, float scale, void* workspace,
    size_t workspace_bytes, int cache_format, int dtype, void* stream) {
  using namespace vmps;
  clear_error();
  const char* what = "paged_decode_attention_cache8";
  if (num_seqs < 0 || num_blocks <= 0 || max_blocks_per_seq <= 0) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: bad sizes (num_seqs=%d num_blocks=%d max_blocks=%d)",
                what, num_seqs, num_blocks, max_blocks_per_seq);
  }
  if (max_blocks_per_seq > (1 << 27) - 1) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: max_blocks %d", what, max_blocks_per_seq);
  }
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (cache_format != VMPS_CACHE_INT8 && cache_format != VMPS_CACHE_E4M3) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: cache_format %d", what, cache_format);
  }
  if (block_size != kCachePage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  const size_t need = vmps_paged_decode_cache8_workspace_bytes(num_seqs, n_q, n_kv, head_dim);
  if (!need) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: num_seqs=%d n_q=%d n_kv=%d head_dim=%d not supported (num_seqs <= 4096, "
                "head_dim 64/128, n_kv <= 64, n_q/n_kv whole and at most 16)",
                what, num_seqs, n_q, n_kv, head_dim);
  }
  if (num_seqs == 0) return VMPS_OK;
  if (!out || !q || !codes || !scales || !block_tables || !seq_lens) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  }
  if (!aligned16(q) || (q_row_stride % 8) || !aligned16(out) || !aligned16(codes) ||
      !aligned16(scales)) {
    return fail(VMPS_ERR_ALIGNMENT,
                "%s: q, out, codes and scales must be 16-byte aligned and the row stride of q a "
                "multiple of 8 elements",
                what);
  }
  if (num_seqs > 1 && q_row_stride < static_cast<int64_t>(n_q) * head_dim) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: row stride smaller than a row", what);
  }
  if (!(scale > 0.f) || !(scale < 1e30f)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: scale %g", what, (double)scale);
  }
  if (!workspace || workspace_bytes < need) {
    return fail(VMPS_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, workspace_bytes,
                need);
  }
  if (reinterpret_cast<uintptr_t>(workspace) & 255) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", what);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  Decode8Params p;
  p.out = out;
  p.q = q;
  p.q_stride = q_row_stride;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.max_blocks = max_blocks_per_seq;
  p.n_kv = n_kv;
  p.G = n_q / n_kv;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_decode8<__half, 64>(p, num_seqs, cache_format, s)
                          : launch_decode8<__half, 128>(p, num_seqs, cache_format, s);
  }
  return head_dim == 64 ? launch_decode8<__nv_bfloat16, 64>(p, num_seqs, cache_format, s)
                        : launch_decode8<__nv_bfloat16, 128>(p, num_seqs, cache_format, s);
}
