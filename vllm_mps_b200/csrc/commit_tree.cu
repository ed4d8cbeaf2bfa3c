// Commit of an accepted branch: which drafted tokens of each tree the model
// agrees with, and their K/V moved to the slots they keep.
//
// The drafted nodes of sequence i sit at slots ctx + 0, ctx + 1, ... in node
// order (node 0 is the tree's root, the last token already decided).  The
// model's own choice after node c is target[c].  Walk from the root: go to the
// lowest-numbered child whose token is target[c], stop where there is none.
// The nodes of that walk, path[0] = 0 < path[1] < ..., keep the slots ctx + k.
//
// Bound: the copy reads and writes 2 * n_kv * head_dim elements per moved
// token and layer; the walk is a chain of dependent look-ups, so each block
// first pulls its sequence's tree into shared memory and one warp walks there
// (32 candidates a step).  Every block of a sequence repeats the walk: that
// costs less than a second launch that waits for one walk's result.  Measured:
// 64 trees of up to 26 nodes, 32 layers x 8 kv heads x 128, 12.1 us (4096 CTAs in
// 4.6 waves: shared memory for the largest tree, 36 KB, allows 6 on an SM); one
// tree of 8 nodes, 22 layers, 3.6 us.
//
// Work split.  One thread owns one 16-byte column of one layer's K or V rows
// of one sequence and moves it for the whole path.  A child comes after its
// parent, so path[k] >= k and the slot a thread writes in round k is the
// source of no later round: reading a batch of sources before writing the
// batch's targets, in path order, is a correct in-place move without any
// synchronisation between threads.
#include "vmps_abi_internal.h"
#include "vmps_common.cuh"

namespace vmps {
namespace {

constexpr int kCommitThreads = 128;
constexpr int kCommitMaxTree = 1024;
constexpr int kCommitBatch = 8;  // sources in flight per thread
constexpr int kPage = 16;

struct CommitParams {
  uint4* pool;
  int64_t layer_stride;  // 16-byte units between layers
  const int32_t* block_tables;
  const int32_t* ctx_lens;
  const int32_t* seq_lens;
  const int32_t* cu_tree;
  const int32_t* parents;
  const int32_t* tokens;
  const int64_t* target;
  int32_t* path;
  int32_t* count;
  int64_t* next_token;
  int num_layers, max_blocks, num_blocks, total_nodes, max_tree;
  int row16;  // 16-byte units of one token's K (or V) row of one layer
  int* err;
};

__global__ void __launch_bounds__(kCommitThreads) commit_tree_kernel(const CommitParams p) {
  __shared__ int s_par[kCommitMaxTree];
  __shared__ int s_tok[kCommitMaxTree];
  __shared__ int64_t s_tgt[kCommitMaxTree];
  __shared__ int s_path[kCommitMaxTree];
  __shared__ int64_t s_src[kCommitMaxTree];  // 16-byte units from a layer's start, -1: no slot
  __shared__ int64_t s_dst[kCommitMaxTree];
  __shared__ int s_count;
  __shared__ int s_first;  // first path position whose node moves

  const int seq = blockIdx.y;
  const int tid = threadIdx.x;
  const int ctx = p.ctx_lens[seq];
  int n = p.seq_lens[seq] - ctx;
  const int row0 = p.cu_tree[seq];
  if (n < 0 || ctx < 0) n = 0;
  if (n > p.max_tree || (n > 0 && (row0 < 0 || static_cast<long long>(row0) + n > p.total_nodes))) {
    if (tid == 0 && blockIdx.x == 0) set_error(p.err, kDevErrQueryRange);
    n = 0;
  }
  for (int i = tid; i < n; i += kCommitThreads) {
    s_par[i] = p.parents[row0 + i];
    s_tok[i] = p.tokens[row0 + i];
    s_tgt[i] = p.target[row0 + i];
  }
  __syncthreads();
  if (tid < 32) {
    int cur = 0, k = 0, first = -1;
    if (n > 0) {
      if (tid == 0) s_path[0] = 0;
      k = 1;
      // Children come after their parent, so the search starts behind it and
      // the walk ends after at most n steps.
      for (int base = 1; base < n;) {
        const int i = base + tid;
        const bool hit = i < n && s_par[i] == cur && s_tok[i] == s_tgt[cur];
        const unsigned m = __ballot_sync(0xffffffffu, hit);
        if (m) {
          cur = base + __ffs(m) - 1;
          if (tid == 0) s_path[k] = cur;
          if (first < 0 && cur != k) first = k;
          ++k;
          base = cur + 1;
        } else {
          base += 32;
        }
      }
    }
    if (tid == 0) {
      s_count = k;
      s_first = first < 0 ? k : first;
      if (blockIdx.x == 0) {
        p.count[seq] = k;
        p.next_token[seq] = n > 0 ? s_tgt[cur] : -1;
      }
    }
  }
  __syncthreads();
  const int count = s_count, first = s_first;
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.max_tree; i += kCommitThreads) {
      p.path[static_cast<size_t>(seq) * p.max_tree + i] = i < count ? s_path[i] : -1;
    }
  }
  if (first >= count) return;  // the branch already sits where it belongs

  auto slot_at = [&](int pos) -> int64_t {
    const int page = pos / kPage;
    if (page >= p.max_blocks) {
      set_error(p.err, kDevErrSeqLen);
      return -1;
    }
    const int b = p.block_tables[static_cast<size_t>(seq) * p.max_blocks + page];
    if (b < 0 || b >= p.num_blocks) {
      set_error(p.err, kDevErrBlockRange);
      return -1;
    }
    return (static_cast<int64_t>(b) * 2 * kPage + pos % kPage) * p.row16;
  };
  for (int i = first + tid; i < count; i += kCommitThreads) {
    s_src[i] = slot_at(ctx + s_path[i]);
    s_dst[i] = slot_at(ctx + i);
  }
  __syncthreads();
  const int per_layer = 2 * p.row16;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kCommitThreads + tid;
  const int layer = static_cast<int>(item / per_layer);
  if (layer >= p.num_layers) return;
  const int e = static_cast<int>(item - static_cast<int64_t>(layer) * per_layer);
  const int is_v = e >= p.row16;
  uint4* base = p.pool + layer * p.layer_stride +
                (is_v ? static_cast<int64_t>(kPage) * p.row16 + e - p.row16 : e);
  for (int k0 = first; k0 < count; k0 += kCommitBatch) {
    uint4 v[kCommitBatch];
#pragma unroll
    for (int j = 0; j < kCommitBatch; ++j) {
      const int k = k0 + j;
      if (k < count && s_src[k] >= 0) v[j] = base[s_src[k]];
    }
#pragma unroll
    for (int j = 0; j < kCommitBatch; ++j) {
      const int k = k0 + j;
      if (k < count && s_src[k] >= 0 && s_dst[k] >= 0) base[s_dst[k]] = v[j];
    }
  }
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" int vmps_commit_tree(int32_t* path, int32_t* count, int64_t* next_token, void* pool,
                                int num_layers, const int32_t* block_tables,
                                int max_blocks_per_seq, const int32_t* ctx_lens,
                                const int32_t* seq_lens, const int32_t* cu_tree,
                                const int32_t* parents, const int32_t* tokens,
                                const int64_t* target_ids, int num_seqs, int total_nodes,
                                int max_tree, int n_kv, int head_dim, int block_size,
                                int num_blocks, int dtype, void* stream) {
  const char* what = "commit_tree";
  clear_error();
  if (num_seqs < 0 || num_layers <= 0 || total_nodes < 0 || max_tree <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0 || n_kv <= 0 || head_dim <= 0) {
    return fail(VMPS_ERR_INVALID_ARG,
                "%s: bad sizes (num_seqs=%d num_layers=%d total_nodes=%d max_tree=%d num_blocks=%d "
                "max_blocks=%d n_kv=%d head_dim=%d)",
                what, num_seqs, num_layers, total_nodes, max_tree, num_blocks, max_blocks_per_seq,
                n_kv, head_dim);
  }
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (block_size != kPage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  if (max_tree > kCommitMaxTree || num_seqs > 65535 ||
      (static_cast<int64_t>(n_kv) * head_dim) % 8 || static_cast<int64_t>(n_kv) * head_dim > 65536) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: max_tree=%d num_seqs=%d n_kv=%d head_dim=%d (max_tree <= %d, num_seqs <= "
                "65535, n_kv * head_dim a multiple of 8 up to 65536)",
                what, max_tree, num_seqs, n_kv, head_dim, kCommitMaxTree);
  }
  if (num_seqs == 0) return VMPS_OK;
  if (!path || !count || !next_token || !pool || !block_tables || !ctx_lens || !seq_lens ||
      !cu_tree || (total_nodes > 0 && (!parents || !tokens || !target_ids))) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  }
  if (!aligned16(pool)) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: pool must be 16-byte aligned", what);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  CommitParams p;
  p.pool = static_cast<uint4*>(pool);
  p.row16 = n_kv * head_dim / 8;
  p.layer_stride = static_cast<int64_t>(num_blocks) * 2 * kPage * p.row16;
  p.block_tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.seq_lens = seq_lens;
  p.cu_tree = cu_tree;
  p.parents = parents;
  p.tokens = tokens;
  p.target = target_ids;
  p.path = path;
  p.count = count;
  p.next_token = next_token;
  p.num_layers = num_layers;
  p.max_blocks = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.total_nodes = total_nodes;
  p.max_tree = max_tree;
  p.err = err;
  const int64_t items = static_cast<int64_t>(num_layers) * 2 * p.row16;
  const int64_t blocks = (items + kCommitThreads - 1) / kCommitThreads;
  if (blocks > 0x7fffffff) return fail(VMPS_ERR_UNSUPPORTED, "%s: too many layers", what);
  commit_tree_kernel<<<dim3(static_cast<unsigned>(blocks), num_seqs), kCommitThreads, 0,
                       static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch(what);
}
