// Paged attention of drafted tree tokens over a sequence's cache.
//
// Row r of sequence i (one drafted token, one query head) sees every cached
// slot t < ctx_lens[i] and the drafted slots ctx_lens[i] + j whose bit j is
// set in its mask row:
//     s_t = scale * q . K_t,   out = sum_t e^(s_t - m) V_t / sum_t e^(s_t - m).
// A row that sees no slot is zero.  Slots that no row may see (past the
// sequence's end) and drafted slots outside a row's mask take no part,
// whatever their bits (a product with their stale values is never formed).
//
// One warp per (row, query head): 32 keys a step, one per lane for the
// scores, then the lanes split head_dim for P . V.
#include "vmps_abi_internal.h"
#include "vmps_common.cuh"

namespace vmps {
namespace {

constexpr int kTreeWarps = 4;
constexpr int kPage = 16;

struct TreeParams {
  void* out;
  const void* q;
  int64_t q_stride;
  const void* pool;
  const int32_t* block_tables;
  const int32_t* ctx_lens;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  const int32_t* cu_q;
  const uint32_t* mask;
  int mask_words, max_blocks, total_q, max_q_len, n_q, n_kv, G, num_blocks;
  float scale_log2;
  int* err;
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kTreeWarps) tree_kernel(const TreeParams p) {
  __shared__ float s_q[kTreeWarps][D];
  const int seq = blockIdx.z, r = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x * kTreeWarps + warp;
  const int q_len = p.q_lens[seq], row0 = p.cu_q[seq];
  if (r >= q_len || head >= p.n_q) return;
  if (row0 < 0 || static_cast<long long>(row0) + q_len > p.total_q || q_len > p.max_q_len) {
    if (lane == 0) set_error(p.err, kDevErrQueryRange);
    if (row0 < 0 || static_cast<long long>(row0) + q_len > p.total_q) return;
  }
  const int row = row0 + r;
  int n = p.seq_lens[seq];
  if (n > p.max_blocks * kPage) {
    if (lane == 0) set_error(p.err, kDevErrSeqLen);
    n = p.max_blocks * kPage;
  }
  const int ctx = min(max(p.ctx_lens[seq], 0), max(n, 0));
  const T* q = static_cast<const T*>(p.q) + row * p.q_stride + static_cast<int64_t>(head) * D;
  for (int d = lane; d < D; d += 32) s_q[warp][d] = Elt<T>::to_f(q[d]);
  __syncwarp();
  const T* pool = static_cast<const T*>(p.pool);
  const int64_t tok = static_cast<int64_t>(p.n_kv) * D;
  const int kvh = head / p.G;
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  for (int t0 = 0; t0 < n; t0 += 32) {
    const int t = t0 + lane;
    bool see = t < n;
    if (see && t >= ctx) {
      const int j = t - ctx;
      see = (j >> 5) < p.mask_words &&
            ((p.mask[static_cast<int64_t>(row) * p.mask_words + (j >> 5)] >> (j & 31)) & 1u);
    }
    int blk = -1;
    if (see) {
      blk = p.block_tables[static_cast<int64_t>(seq) * p.max_blocks + t / kPage];
      if (blk < 0 || blk >= p.num_blocks) {
        set_error(p.err, kDevErrBlockRange);
        blk = -1;
      }
    }
    float s = -INFINITY;
    const int64_t at = ((static_cast<int64_t>(blk) * 2) * kPage + t % kPage) * tok + kvh * D;
    if (see) {
      s = 0.f;
      if (blk >= 0) {
        for (int d = 0; d < D; ++d) s += s_q[warp][d] * Elt<T>::to_f(pool[at + d]);
      }
      s *= p.scale_log2;
    }
    float mx = s;
    for (int sh = 16; sh; sh >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
    const float mn = fmaxf(m, mx);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float al = exp2f(m - base);
    const float e = see ? exp2f(s - base) : 0.f;
    m = mn;
    l = l * al + e;
    for (int i = 0; i < D / 32; ++i) o[i] *= al;
    unsigned todo = __ballot_sync(0xffffffffu, see && blk >= 0);
    while (todo) {
      const int j = __ffs(todo) - 1;
      todo &= todo - 1;
      const float pj = __shfl_sync(0xffffffffu, e, j);
      const int64_t vat = __shfl_sync(0xffffffffu, at, j) + kPage * tok;
      for (int i = 0; i < D / 32; ++i) o[i] += pj * Elt<T>::to_f(pool[vat + i * 32 + lane]);
    }
  }
  for (int sh = 16; sh; sh >>= 1) l += __shfl_xor_sync(0xffffffffu, l, sh);
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(row) * p.n_q + head) * D;
  for (int i = 0; i < D / 32; ++i) out[i * 32 + lane] = Elt<T>::from_f(o[i] * inv);
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" size_t vmps_paged_tree_attention_workspace_bytes(int num_seqs, int max_q_len, int n_q,
                                                            int n_kv, int head_dim, int dtype) {
  (void)num_seqs, (void)max_q_len, (void)n_q, (void)n_kv, (void)head_dim, (void)dtype;
  return 256;
}

extern "C" int vmps_paged_tree_attention(
    void* out, const void* q, int64_t q_row_stride, const void* pool, const int32_t* block_tables,
    int max_blocks_per_seq, const int32_t* ctx_lens, const int32_t* seq_lens,
    const int32_t* q_lens, const int32_t* cu_q, const int32_t* tree_mask, int mask_words,
    int num_seqs, int total_q, int max_q_len, int n_q, int n_kv, int head_dim, int block_size,
    int num_blocks, float scale, void* workspace, size_t workspace_bytes, int dtype,
    void* stream) {
  const char* what = "paged_tree_attention";
  clear_error();
  if (num_seqs < 0 || total_q < 0 || max_q_len < 0 || mask_words <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0) {
    return fail(VMPS_ERR_INVALID_ARG,
                "%s: bad sizes (num_seqs=%d total_q=%d max_q_len=%d mask_words=%d num_blocks=%d "
                "max_blocks=%d)",
                what, num_seqs, total_q, max_q_len, mask_words, num_blocks, max_blocks_per_seq);
  }
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (block_size != kPage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  if ((head_dim != 64 && head_dim != 128) || n_kv <= 0 || n_kv > 64 || n_q <= 0 || n_q % n_kv ||
      n_q / n_kv > 16) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: n_q=%d n_kv=%d head_dim=%d not supported (head_dim 64/128, n_kv <= 64, "
                "n_q/n_kv a whole number up to 16)",
                what, n_q, n_kv, head_dim);
  }
  if (num_seqs > 4096 || max_q_len > 65535 || max_blocks_per_seq > (1 << 26)) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: num_seqs %d > 4096, max_q_len %d > 65535 or max_blocks %d",
                what, num_seqs, max_q_len, max_blocks_per_seq);
  }
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return VMPS_OK;
  if (!out || !q || !pool || !block_tables || !ctx_lens || !seq_lens || !q_lens || !cu_q ||
      !tree_mask) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  }
  if (!aligned16(pool) || !aligned16(q) || !aligned16(out) || (q_row_stride % 8)) {
    return fail(VMPS_ERR_ALIGNMENT,
                "%s: pool/q/out must be 16-byte aligned and the q row stride a multiple of 8 "
                "elements",
                what);
  }
  if (q_row_stride < static_cast<int64_t>(n_q) * head_dim) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: q row stride smaller than a row", what);
  }
  if (!(scale > 0.f) || !(scale < 1e30f)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: scale %g", what, (double)scale);
  }
  if (!workspace || workspace_bytes < 256) {
    return fail(VMPS_ERR_WORKSPACE, "%s: workspace %zu bytes < %d needed", what, workspace_bytes, 256);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  TreeParams p;
  p.out = out;
  p.q = q;
  p.q_stride = q_row_stride;
  p.pool = pool;
  p.block_tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.seq_lens = seq_lens;
  p.q_lens = q_lens;
  p.cu_q = cu_q;
  p.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  p.mask_words = mask_words;
  p.max_blocks = max_blocks_per_seq;
  p.total_q = total_q;
  p.max_q_len = max_q_len;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.G = n_q / n_kv;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = err;
  const dim3 grid((n_q + kTreeWarps - 1) / kTreeWarps, max_q_len, num_seqs);
  const dim3 block(32 * kTreeWarps);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    if (head_dim == 64) tree_kernel<__half, 64><<<grid, block, 0, s>>>(p);
    else tree_kernel<__half, 128><<<grid, block, 0, s>>>(p);
  } else {
    if (head_dim == 64) tree_kernel<__nv_bfloat16, 64><<<grid, block, 0, s>>>(p);
    else tree_kernel<__nv_bfloat16, 128><<<grid, block, 0, s>>>(p);
  }
  return check_launch(what);
}
