// Kernel 10: pages of the 8-bit cache read back into 16-bit pages.
//
//   pool[dst][kv][t][h][d] = round(code * scale)   for the sequence's tokens,
//   0 for the rest of its last page (attention over those pages reads them).
//
// What bounds it: the bytes read and written.
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
  int pages;  // of a sequence per CTA
  int width, rows;  // columns of a page that a CTA takes at a time, and rows of each
  int span;         // rows of a page that are a CTA's
  bool wide;        // 32-byte aligned pool
  int* err;
};

constexpr int kReadThreads = 256;
constexpr int kReadResident = 6;  // blocks of an SM

// A thread keeps to one 16-byte column of the page's rows (32 of them: K and V of 16
// tokens; n_kv * D codes each), so that nothing is divided per row, and stores a whole
// 32-byte sector (with two 16-byte stores, half a sector of every lane each, 131071 tokens of
// 8 heads x 128 took 150 us).  What hides the loads is the number of blocks: those tokens take
// 131 us (6.2 TB/s read and written), with four rows' loads in flight per thread, and fewer
// blocks, 160.
template <typename T, int D, typename Code>
__global__ void __launch_bounds__(kReadThreads, kReadResident) read_cache8_kernel(const ReadParams p) {
  chain_link();
  const int s = blockIdx.y;
  const int len = p.seq_lens[s];
  const int page0 = blockIdx.x * p.pages;
  if (len <= 0 || page0 > (len - 1) / kCachePage) return;
  int page1 = min(page0 + p.pages, (len - 1) / kCachePage + 1);
  if (page1 > p.max_blocks) page1 = p.max_blocks;
  if ((len - 1) / kCachePage >= p.max_blocks && blockIdx.x == 0 && threadIdx.x == 0) {
    set_error(p.err, kDevErrSeqLen);
  }
  const int row_codes = p.n_kv * D;
  const int columns = row_codes / 16;
  const int width = p.width, rows = p.rows;
  const int c0 = threadIdx.x % width, r0 = threadIdx.x / width;
  if (r0 >= rows) return;
  const int ra = blockIdx.z * p.span + r0, rb = blockIdx.z * p.span + p.span;
  for (int page = page0; page < page1; ++page) {
    const int64_t at = static_cast<int64_t>(s) * p.max_blocks + page;
    const int src = p.block_tables[at], dst = p.dst_tables[at];
    if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.pool_blocks) {
      if (threadIdx.x == 0) set_error(p.err, kDevErrBlockRange);
      continue;
    }
    const int live = len - page * kCachePage;  // tokens from this page on
    for (int c = c0; c < columns; c += width) {
      const int64_t block = static_cast<int64_t>(2 * kCachePage) * row_codes;
      const uint8_t* codes = p.codes + src * block + c * 16;
      const float* scales =
          p.scales + (static_cast<int64_t>(src) * p.n_kv + c * 16 / D) * 2 * kCachePage;
      T* out = static_cast<T*>(p.pool) + dst * block + c * 16;
#pragma unroll 1
      for (int r = ra; r < rb; r += rows) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);  // K's 16 tokens, then V's: the scales' order too
        float sc = 0.f;
        if (r % kCachePage < live) {
          w = __ldcs(reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(r) * row_codes));
          sc = scales[r];
        }
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[4];
          Code::unpack4(v[i], x);
          o[2 * i] = Elt<T>::pack(x[0] * sc, x[1] * sc);
          o[2 * i + 1] = Elt<T>::pack(x[2] * sc, x[3] * sc);
        }
        T* row = out + static_cast<int64_t>(r) * row_codes;
        if (p.wide) {
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row),
                       "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]),
                       "r"(o[7])
                       : "memory");
        } else {
          *reinterpret_cast<uint4*>(row) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(row + 8) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
    }
  }
}

template <typename T, int D>
int launch_read(ReadParams p, int num_seqs, int format, cudaStream_t s) {
  // One page a CTA, more where the tables are wide: a CTA without pages costs a launch slot.
  const int64_t all = static_cast<int64_t>(p.max_blocks) * num_seqs;
  p.pages = static_cast<int>((all + 16383) / 16384);
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  // Equal passes over the columns (40 heads x 128, 16384 tokens 102 -> 91 us).
  const int columns = p.n_kv * D / 16, passes = (columns + kReadThreads - 1) / kReadThreads;
  p.width = (columns + passes - 1) / passes;
  p.rows = kReadThreads / p.width;
  // Few pages are shared out by rows while every thread keeps one, to 2048 CTAs: 8 heads x
  // 128, 4 pages 4.1 -> 1.8 us, 64 pages 4.8 -> 3.1, 512 pages 12.5 -> 11.4 (12.1 with 4096
  // CTAs); 64 heads, 13 pages 22.2 -> 3.4; 131071 tokens, however, 131 -> 137.
  p.span = 2 * kCachePage;
  for (int split = 2; p.rows <= p.span / 2 && all * split <= 2048; split *= 2) p.span /= 2;
  const dim3 grid((p.max_blocks + p.pages - 1) / p.pages, num_seqs, 2 * kCachePage / p.span);
  // An early start saves small calls half a microsecond, but the blocks of larger grids
  // are then spread unevenly over the SMs that the launch before still holds (512 pages of
  // 8 heads x 128, undivided: 13 -> 17 us).
  const bool early = static_cast<int64_t>(grid.x) * grid.y * grid.z <= sms;
  const cudaError_t e =
      format == VMPS_CACHE_INT8
          ? launch_link(read_cache8_kernel<T, D, Int8Code>, early, grid, dim3(kReadThreads), 0, s, p)
          : launch_link(read_cache8_kernel<T, D, E4m3Code>, early, grid, dim3(kReadThreads), 0, s, p);
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "read_cache8: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
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
  ReadParams p = {};
  p.pool = pool;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.block_tables = block_tables;
  p.dst_tables = dst_tables;
  p.seq_lens = seq_lens;
  p.max_blocks = max_blocks_per_seq;
  p.n_kv = n_kv;
  p.num_blocks = num_blocks;
  p.pool_blocks = pool_blocks;
  p.wide = (reinterpret_cast<uintptr_t>(pool) & 31) == 0;
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_read<__half, 64>(p, num_seqs, cache_format, s)
                          : launch_read<__half, 128>(p, num_seqs, cache_format, s);
  }
  return head_dim == 64 ? launch_read<__nv_bfloat16, 64>(p, num_seqs, cache_format, s)
                        : launch_read<__nv_bfloat16, 128>(p, num_seqs, cache_format, s);
}

extern "C" int vmps_read_cache8_args(const vmps_read_args* a, void* stream) {
  if (!a) return vmps::fail(VMPS_ERR_INVALID_ARG, "read_cache8: NULL arguments");
  return vmps_read_cache8(a->pool, a->pool_blocks, a->dst_tables, a->codes, a->scales,
                          a->block_tables, a->max_blocks_per_seq, a->seq_lens, a->num_seqs, a->n_kv,
                          a->head_dim, a->block_size, a->num_blocks, a->cache_format, a->dtype,
                          stream);
}
