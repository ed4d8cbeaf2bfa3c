// Kernel 10: pages of the 8-bit cache read back into 16-bit pages.
//
//   pool[dst][kv][t][h][d] = round(code * scale)   for the sequence's tokens,
//   0 for the rest of its last page (attention over those pages reads them).
#include "cache8.cuh"
#include "vmps_abi_internal.h"

namespace vmps {
namespace {

struct ReadParams {
  void* pool;
  const uint8_t* codes;
  const float* scales;
  const int32_t* block_tables;
  const int32_t* dst_tables;
  const int32_t* seq_lens;
  int max_blocks, n_kv, num_blocks, pool_blocks;
  int* err;
};

template <typename T, int D, typename Code>
__global__ void __launch_bounds__(256) read_cache8_kernel(const ReadParams p) {
  const int s = blockIdx.y;
  const int page = blockIdx.x;
  const int len = p.seq_lens[s];
  if (len <= 0 || page > (len - 1) / kCachePage) return;
  if ((len - 1) / kCachePage >= p.max_blocks && page == 0 && threadIdx.x == 0) {
    set_error(p.err, kDevErrSeqLen);
  }
  const int64_t at = static_cast<int64_t>(s) * p.max_blocks + page;
  const int src = p.block_tables[at], dst = p.dst_tables[at];
  if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.pool_blocks) {
    if (threadIdx.x == 0) set_error(p.err, kDevErrBlockRange);
    return;
  }
  const int per_kind = kCachePage * p.n_kv * D;
  const int live = len - page * kCachePage;  // tokens of this page
  const uint8_t* codes = p.codes + static_cast<int64_t>(src) * 2 * per_kind;
  const float* scales = p.scales + static_cast<int64_t>(src) * 2 * p.n_kv * kCachePage;
  T* out = static_cast<T*>(p.pool) + static_cast<int64_t>(dst) * 2 * per_kind;
  for (int e = threadIdx.x * 8; e < 2 * per_kind; e += blockDim.x * 8) {
    const int kind = e >= per_kind;
    const int row = (e - kind * per_kind) / D;  // token * n_kv + head
    const int t = row / p.n_kv, h = row % p.n_kv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t < live) {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + e);
      const float sc = scales[(h * 2 + kind) * kCachePage + t];
      float a[4], b[4];
      Code::unpack4(w.x, a);
      Code::unpack4(w.y, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i] * sc;
        x[4 + i] = b[i] * sc;
      }
    }
    *reinterpret_cast<uint4*>(out + e) =
        make_uint4(Elt<T>::pack(x[0], x[1]), Elt<T>::pack(x[2], x[3]), Elt<T>::pack(x[4], x[5]),
                   Elt<T>::pack(x[6], x[7]));
  }
}

template <typename T, int D>
int launch_read(const ReadParams& p, int num_seqs, int format, cudaStream_t s) {
  const dim3 grid(p.max_blocks, num_seqs);
  if (format == VMPS_CACHE_INT8) {
    read_cache8_kernel<T, D, Int8Code><<<grid, 256, 0, s>>>(p);
  } else {
    read_cache8_kernel<T, D, E4m3Code><<<grid, 256, 0, s>>>(p);
  }
  return check_launch("read_cache8");
}

}  // namespace
}  // namespace vmps

extern "C" int vmps_read_cache8(void* pool, int pool_blocks, const int32_t* dst_tables,
                                const void* codes, const float* scales,
                                const int32_t* block_tables, int max_blocks_per_seq,
                                const int32_t* seq_lens, int num_seqs, int n_kv, int head_dim,
                                int block_size, int num_blocks, int cache_format, int dtype,
                                void* stream) {
  using namespace vmps;
  clear_error();
  const char* what = "read_cache8";
  if (num_seqs < 0 || n_kv <= 0 || n_kv > 64 || num_blocks <= 0 || pool_blocks <= 0 ||
      max_blocks_per_seq <= 0) {
    return fail(VMPS_ERR_INVALID_ARG,
                "%s: bad sizes (num_seqs=%d n_kv=%d num_blocks=%d pool_blocks=%d max_blocks=%d)",
                what, num_seqs, n_kv, num_blocks, pool_blocks, max_blocks_per_seq);
  }
  if (num_seqs > 4096) return fail(VMPS_ERR_UNSUPPORTED, "%s: num_seqs %d > 4096", what, num_seqs);
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (cache_format != VMPS_CACHE_INT8 && cache_format != VMPS_CACHE_E4M3) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: cache_format %d", what, cache_format);
  }
  if (head_dim != 64 && head_dim != 128) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  }
  if (block_size != kCachePage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  if (num_seqs == 0) return VMPS_OK;
  if (!pool || !dst_tables || !codes || !scales || !block_tables || !seq_lens) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  }
  if (!aligned16(pool) || !aligned16(codes) || !aligned16(scales)) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: pool, codes and scales must be 16-byte aligned", what);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  ReadParams p{pool,     static_cast<const uint8_t*>(codes), scales, block_tables, dst_tables,
               seq_lens, max_blocks_per_seq,                 n_kv,   num_blocks,   pool_blocks,
               err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_read<__half, 64>(p, num_seqs, cache_format, s)
                          : launch_read<__half, 128>(p, num_seqs, cache_format, s);
  }
  return head_dim == 64 ? launch_read<__nv_bfloat16, 64>(p, num_seqs, cache_format, s)
                        : launch_read<__nv_bfloat16, 128>(p, num_seqs, cache_format, s);
}
