/*
 * vmps.h -- C ABI of libvmps_kernels.so, the sm_100a (B200) kernels behind
 * the paged decode-attention step of vllm_mps.
 *
 * The reference (Nihar0071/vllm_mps) has no C ABI: its device code is two
 * Metal shaders held as Python strings and its CPU path is PyTorch code.
 * Each entry point below names the reference interface it replaces.  The
 * Python side binds these symbols with ctypes (vllm_mps_b200/kernels).
 *
 * Conventions shared by every entry point:
 *   - All pointers are device pointers unless stated; the caller owns every
 *     buffer.  The library allocates nothing; besides the device error word
 *     it keeps one fixed scratch array in its own device memory, used only
 *     by vmps_paged_decode_attention_noalloc (its calls must not overlap on
 *     the GPU).
 *   - `stream` is a cudaStream_t (NULL = legacy default stream).  Work is
 *     only enqueued; calls return before the GPU finishes.
 *   - `dtype` is VMPS_DTYPE_F16 or VMPS_DTYPE_BF16 for every 16-bit tensor
 *     of the call (q, k, v, pool, out).
 *   - The KV pool has the reference layout
 *       pool[num_blocks][2][block_size][n_kv][head_dim]   (dim 1: 0 = K, 1 = V)
 *     (memory/mps_memory_pool.py:62-66), contiguous.
 *   - Return 0 on success or a negative VMPS_ERR_* code; vmps_last_error()
 *     then describes the failure (thread-local).  Arguments are checked on
 *     the host before anything is launched.  Device-side index violations
 *     skip the access and set a bit in the error word (vmps_debug_error_word).
 */
#ifndef VMPS_H_
#define VMPS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VMPS_OK 0
#define VMPS_ERR_INVALID_ARG (-1)  /* bad pointer, size or shape */
#define VMPS_ERR_UNSUPPORTED (-2)  /* valid but not built (e.g. head_dim 96) */
#define VMPS_ERR_ALIGNMENT (-3)    /* a pointer or stride is not 16-byte aligned */
#define VMPS_ERR_WORKSPACE (-4)    /* workspace missing or too small */
#define VMPS_ERR_CUDA (-5)         /* CUDA runtime/driver error */

#define VMPS_DTYPE_F16 0
#define VMPS_DTYPE_BF16 1

#define VMPS_CACHE_16BIT 0 /* the pool in the call's dtype */
#define VMPS_CACHE_INT8 1  /* 8-bit cache of int8 codes */
#define VMPS_CACHE_E4M3 2  /* 8-bit cache of e4m3 codes */

/* Library version string, e.g. "vmps 0.1.0 sm_100a". */
const char* vmps_version(void);

/* Description of the last failure on the calling thread ("" if none). */
const char* vmps_last_error(void);

/*
 * Fused RoPE + reshape-and-cache (kernel 1).
 *
 * Replaces the per-sequence RoPE loop and K/V write loop of
 * PagedAttentionLayer._forward_batch (layers/paged_attention_layer.py:275-286
 * and :317-324), i.e. RotaryEmbedding.forward (layers/rotary_embedding.py:55-76)
 * followed by MPSMemoryPool.write_kv (memory/mps_memory_pool.py:82-102), and
 * Phase 1 of the Metal fused_attention shader (kernels/__init__.py:139-161).
 *
 * For each sequence i in [0, num_seqs):
 *   q_out[i] = rope(q[i], positions[i])                  (n_q heads)
 *   pool[slot / block_size][0][slot % block_size] = rope(k[i], positions[i])
 *   pool[slot / block_size][1][slot % block_size] = v[i]
 * with slot = slot_mapping[i] (= block_table[pos / block_size] * block_size
 * + pos % block_size); a negative slot skips the write.  rope() is the
 * rotate-half form with cos/sin = cos/sin(position * inv_freq[j]) rounded
 * to the model dtype and each product and the sum rounded to the model
 * dtype, as the reference computes it.  inv_freq (head_dim/2 floats) = NULL
 * means "no rotation" (K/V are written as given, q_out = q).
 *
 * q/k/v rows are head-major [heads][head_dim] with a row stride in elements
 * between sequences (so slices of a fused QKV output work).  q_out may equal
 * q (in-place) and uses q_row_stride too.  positions and slot_mapping are
 * int32[num_seqs] on the device.
 */
int vmps_rope_reshape_and_cache(void* q_out, const void* q, int64_t q_row_stride,
                                const void* k, int64_t k_row_stride, const void* v,
                                int64_t v_row_stride, const int32_t* positions,
                                const int32_t* slot_mapping, const float* inv_freq, void* pool,
                                int num_seqs, int n_q, int n_kv, int head_dim, int block_size,
                                int num_blocks, int dtype, void* stream);

/*
 * Workspace needed by vmps_paged_decode_attention / vmps_paged_decode_step
 * on the current device for up to `num_seqs` sequences: split-K partial
 * results of sequences cut between CTAs, and one arrival counter per kv head
 * and sequence (a fixed 1 MiB region, so one workspace serves calls of any
 * shape).  The workspace must be zero-filled once after allocation
 * (vmps_paged_decode_workspace_init); every call leaves the counters at zero
 * again.  Calls sharing a workspace must be ordered (same stream).  Returns 0
 * if the shape is unsupported.
 */
size_t vmps_paged_decode_workspace_bytes(int num_seqs, int n_q, int n_kv, int head_dim,
                                         int dtype);

/* cudaMemsetAsync(workspace, 0, bytes, stream): the one-time initialisation
 * a new workspace needs. */
int vmps_paged_decode_workspace_init(void* workspace, size_t workspace_bytes, void* stream);

/*
 * Paged decode attention (kernel 2), one query token per sequence.
 *
 * Replaces the gather/pad loop, GQA expansion and masked softmax attention of
 * PagedAttentionLayer._forward_batch (layers/paged_attention_layer.py:326-359),
 * MPSMemoryPool.gather_blocks_tensor (memory/mps_memory_pool.py:159-176), and
 * Phases 2-4 of the Metal fused_attention shader (kernels/__init__.py:166-241).
 *
 *   out[i][h][:] = softmax_t( scale * q[i][h] . K_i[t][h / G] ) . V_i[t][h / G]
 * for t < seq_lens[i], G = n_q / n_kv, where K_i[t] / V_i[t] is slot
 * t % block_size of block block_tables[i * max_blocks_per_seq + t / block_size].
 * Computed with fp32 scores, fp32 online softmax and fp32 accumulation;
 * out is rounded once to the model dtype.  q and out are [num_seqs][n_q][head_dim]
 * contiguous (q and the pool 16-byte aligned, out 2-byte aligned:
 * VMPS_ERR_ALIGNMENT otherwise); seq_lens counts the new token; block tables are int32, only
 * the first ceil(seq_len / block_size) entries of a row are read.  A
 * sequence with seq_len 0 gets a zero output row.
 *
 * Supported: head_dim 64 or 128, block_size 16, n_q / n_kv in {1,2,4,8,16},
 * n_kv <= 64, num_seqs <= 4096.  Long sequences are split across CTAs (flash-decoding)
 * and the last piece to finish merges them in the same launch.  The kernel
 * is launched with programmatic dependent launch (it waits for the
 * preceding kernel's writes before reading anything).
 */
int vmps_paged_decode_attention(void* out, const void* q, const void* pool,
                                const int32_t* block_tables, int max_blocks_per_seq,
                                const int32_t* seq_lens, int num_seqs, int n_q, int n_kv,
                                int head_dim, int block_size, int num_blocks, float scale,
                                void* workspace, size_t workspace_bytes, int dtype, void* stream);

/*
 * One decode step of one attention layer in a single kernel launch.
 *
 * Same result as vmps_rope_reshape_and_cache (rotated K and V written to
 * the pool slot) followed by vmps_paged_decode_attention on the rotated q,
 * i.e. PagedAttentionLayer's batched step between its projections
 * (layers/paged_attention_layer.py:275-359) and the whole Metal
 * fused_attention shader (kernels/__init__.py:99-242) with RoPE folded in.
 * q is rotated in registers and left unchanged in memory.  Requirements:
 * seq_lens[i] >= 1 and slot_mapping[i] addresses a slot of the last page of
 * sequence i (as the reference's write_info always does for position
 * seq_len-1); otherwise the write is flagged in the error word (bit 32).
 * The launch may start while the kernel before it on the stream still runs
 * (programmatic dependent launch): the step metadata -- seq_lens, block
 * tables, positions, slot_mapping, inv_freq -- is read before that kernel
 * finishes, so it must not produce them (pool pages are only pulled into L2
 * then, which is coherent with its writes); q/k/v and the pool contents are
 * read after it finishes.
 * q/k/v rows may have any row stride (slices of a fused QKV output).
 */
int vmps_paged_decode_step(void* out, void* q, int64_t q_row_stride, const void* k,
                           int64_t k_row_stride, const void* v, int64_t v_row_stride,
                           const int32_t* positions, const int32_t* slot_mapping,
                           const float* inv_freq, void* pool, const int32_t* block_tables,
                           int max_blocks_per_seq, const int32_t* seq_lens, int num_seqs, int n_q,
                           int n_kv, int head_dim, int block_size, int num_blocks, float scale,
                           void* workspace, size_t workspace_bytes, int dtype, void* stream);

/*
 * Allocation-free variant of vmps_paged_decode_attention.  No counterpart in
 * the reference.  It exists for callers that cannot allocate device memory
 * while running (a C/FFI host without a caching allocator, or a process that
 * has already reserved all free HBM for its KV pool), which therefore cannot
 * pass the workspace the other entry point needs.
 *
 * Same arguments and results as vmps_paged_decode_attention minus the
 * workspace: the split-K scratch is a fixed 8 MiB device array inside the
 * library, held on every GPU that loads the library until exit.  Calls that
 * would need more scratch (vmps_paged_decode_workspace_bytes) return
 * VMPS_ERR_WORKSPACE; on a 148-SM B200 every supported shape with up to 8
 * query heads per kv head fits, 16 query heads per kv head does not.  All calls
 * on a device share the array, so calls that may overlap on the GPU race and
 * must be ordered on one stream.  Every call first clears the merge counters
 * it uses (n_kv * num_seqs ints) with a cudaMemsetAsync on `stream`, so a
 * call that gave up a bounded wait (error bit 8) cannot disturb the next.
 * The first call on a device looks up the array's address
 * (cudaGetSymbolAddress) and caches it; make that first call before any
 * stream capture.  Allocates nothing (no cudaMalloc/cudaFree).
 */
int vmps_paged_decode_attention_noalloc(void* out, const void* q, const void* pool,
                                        const int32_t* block_tables, int max_blocks_per_seq,
                                        const int32_t* seq_lens, int num_seqs, int n_q, int n_kv,
                                        int head_dim, int block_size, int num_blocks, float scale,
                                        int dtype, void* stream);

/*
 * Causal paged prefill attention (kernel 3, tcgen05 tensor cores).  Replaces
 * the reference's prompt processing, which runs the single-token path once
 * per prompt token (layers/paged_attention_layer.py:175-241, driven by
 * benchmarks/batch_size_benchmark.py:49-60): row r of sequence i sits at
 * position q_start_pos[i] + r and attends to the sequence's slots
 * 0..q_start_pos[i] + r, which must already hold K/V (written by
 * vmps_rope_reshape_and_cache for the new rows).
 *
 * q:    [total_q rows][n_q][head_dim], rotated (kernel 1's q_out), row r of
 *       sequence i at cu_q[i] + r; row stride q_row_stride elements
 *       (multiple of 8).  16-byte aligned.
 * out:  [total_q][n_q][head_dim], contiguous, same dtype; rows are written
 *       only for r < q_lens[i].
 * q_start_pos, q_lens, cu_q: int32 [num_seqs] on the device.  max_q_len
 *       bounds q_lens (it sizes the grid; rows past it are not computed and
 *       set error bit 64).
 * block_tables: int32 [num_seqs][max_blocks_per_seq] covering
 *       q_start_pos[i] + q_lens[i] slots.
 * Supported: head_dim 64 or 128, block_size 16, n_q/n_kv in {1,2,4,8,16}.
 * Allocates nothing; no workspace.
 */
int vmps_paged_prefill_attention(void* out, const void* q, int64_t q_row_stride,
                                 const void* pool, const int32_t* block_tables,
                                 int max_blocks_per_seq, const int32_t* q_start_pos,
                                 const int32_t* q_lens, const int32_t* cu_q, int num_seqs,
                                 int total_q, int max_q_len, int n_q, int n_kv, int head_dim,
                                 int block_size, int num_blocks, float scale, int dtype,
                                 void* stream);

/*
 * Element-wise work between the GEMMs of a Llama decoder layer, fused for
 * the CUDA-graph decode step.  No kernel counterpart in the reference, which
 * runs these as HuggingFace modules (LlamaRMSNorm, the residual additions of
 * LlamaDecoderLayer, SiLU(gate) * up of LlamaMLP); the rounding points of
 * those modules are kept.
 *
 * vmps_add_rmsnorm: residual <- residual + delta (delta may be NULL), then
 *   out <- weight * (residual * rsqrt(mean(residual^2) + eps)) for `rows`
 *   rows of `hidden` elements (hidden % 8 == 0; rows 16-byte aligned).
 * vmps_silu_mul: out[:, :inter] <- silu(gate_up[:, :inter]) * gate_up[:, inter:2*inter].
 * vmps_embed_rmsnorm: the step's first kernel (the HF embedding lookup and
 *   the first layer's input LlamaRMSNorm).  Row i's token is prev[src[i]]
 *   when src is non-NULL and src[i] >= 0 (an id the previous step sampled on
 *   the device: a pipelined engine launches step k+1 before it reads step
 *   k's tokens back), else tokens[i]; residual[i] <- table[token] (table:
 *   [vocab, hidden]), out[i] <- RMSNorm(residual[i]) * weight as
 *   vmps_add_rmsnorm with delta NULL.  src[i] >= n_prev or a token outside
 *   [0, vocab) sets error bit 128 and zeroes the row.
 */
int vmps_add_rmsnorm(void* out, int64_t out_row_stride, void* residual, int64_t res_row_stride,
                     const void* delta, int64_t delta_row_stride, const void* weight, int rows,
                     int hidden, float eps, int dtype, void* stream);
int vmps_silu_mul(void* out, int64_t out_row_stride, const void* gate_up,
                  int64_t in_row_stride, int rows, int inter, int dtype, void* stream);
int vmps_embed_rmsnorm(void* out, int64_t out_row_stride, void* residual,
                       int64_t res_row_stride, const void* table, int64_t vocab,
                       const int32_t* tokens, const int32_t* src, const int64_t* prev,
                       int n_prev, const void* weight, int rows, int hidden, float eps,
                       int dtype, void* stream);

/*
 * Decode GEMM for the projections around the attention step at decode batch
 * sizes (replaces the nn.Linear calls of the HF decoder layer that the
 * reference's models/llama_adapter.py:137-207 runs: q/k/v, o, gate/up and
 * down projections).  out[M, N] = x[M, K] . w[N, K]^T, fp32 accumulation,
 * rounded to the 16-bit type.  With silu_mul != 0, w is the fused [gate; up]
 * weight of 2N rows and out[M, N] = silu(x . Wg^T) * (x . Wu^T), each
 * projection rounded first (transformers LlamaMLP).
 * Shapes: M <= 8, N % 8 == 0, K % 64 == 0, K <= 8192; x and w 16-byte
 * aligned, x rows a multiple of 8 elements apart; out 4-byte aligned with an
 * even row stride.  vmps_decode_gemm_supported says whether a shape is
 * built (1) or not (0), so a caller can fall back to its GEMM library.
 * Launched with programmatic dependent launch: the weight stream starts
 * before the wait on the previous kernel in the stream.
 */
int vmps_decode_gemm_supported(int M, int N, int K, int silu_mul);
int vmps_decode_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                     const void* w, int M, int N, int K, int silu_mul, int dtype, void* stream);

/*
 * Batch GEMM for the same projections at decode batch sizes 1..256 (the
 * nn.Linear calls of models/llama_adapter.py:137-207 at the engine's batch;
 * no kernel counterpart in the reference): out[M, N] = x[M, K] . w[N, K]^T,
 * fp16 or bf16, fp32 accumulation on the tcgen05 tensor cores, one rounding.
 * Requires N % 128 == 0, K % 64 == 0, x, w and out 16-byte aligned, x and
 * out rows a multiple of 8 elements apart (x rows at least K, out rows at
 * least N).  Narrow shapes split K over a thread-block cluster of up to 4
 * CTAs whose fp32 partials are summed (in a fixed order) through the
 * caller's workspace: vmps_batch_gemm_split returns that cluster size for a
 * shape on the current device (0 = shape not built) and
 * vmps_batch_gemm_workspace_bytes the workspace it needs (0 = none; at most
 * 16 MiB), which must be 16-byte aligned; it needs no initialisation, and
 * calls that may overlap on the GPU need different workspaces (calls on one
 * stream never overlap).  VMPS_ERR_WORKSPACE if it is missing or too small.
 * Launched with programmatic dependent launch: the weight stream starts
 * before the previous kernel has finished.
 */
int vmps_batch_gemm_split(int M, int N, int K);
size_t vmps_batch_gemm_workspace_bytes(int M, int N, int K, int dtype);
int vmps_batch_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                    const void* w, int M, int N, int K, void* workspace, size_t workspace_bytes,
                    int dtype, void* stream);

/*
 * Attention of drafted tokens (a tree, or any set of drafts) over the paged
 * cache: the check of speculative decoding.  No counterpart in the reference,
 * which decodes one token per pass.
 *
 * Sequence i holds seq_lens[i] slots: ctx_lens[i] cached tokens, then its
 * drafted tokens (draft j at slot ctx_lens[i] + j, K/V already written, e.g.
 * by vmps_rope_reshape_and_cache).  Its query rows are cu_q[i] + r, r <
 * q_lens[i]; a row sees every slot t < ctx_lens[i] and the draft j whose bit
 * (j & 31) of tree_mask[row][j >> 5] is set:
 *   out[row][h] = softmax_t(scale * q[row][h] . K[t][h / G]) . V[t][h / G].
 * Scores, maxima and sums are fp32; a softmax weight is rounded to the 16-bit
 * type for its product with V, the output once.
 * A row that sees no slot is zero.  Slots no row sees and drafts outside a
 * row's mask take no part, whatever they hold (NaN and infinities included).
 * Mask bits of drafts past seq_lens[i] are ignored; drafts past
 * 32 * mask_words are seen by no row.  ctx_lens[i] above seq_lens[i] counts
 * as seq_lens[i].
 *
 * q:    [total_q][n_q][head_dim], rotated, row stride q_row_stride elements
 *       (multiple of 8), 16-byte aligned.  One row per sequence is a decode
 *       step; the last rows of a tree alone are one level of its drafting.
 * out:  [total_q][n_q][head_dim] contiguous, 16-byte aligned; only the rows
 *       of a sequence are written.
 * tree_mask: int32 [total_q][mask_words], contiguous.
 * ctx_lens, seq_lens, q_lens, cu_q: int32 [num_seqs] on the device.
 * max_q_len bounds q_lens (rows past it are not computed and set error bit
 *       64, as do rows outside [0, total_q)).
 * workspace: vmps_paged_tree_attention_workspace_bytes bytes (0: none is
 *       needed, workspace may be NULL), 256-byte aligned, no initialisation;
 *       calls that may overlap on the GPU need different workspaces.  The size
 *       depends on the device and on the arguments given, not on the lengths;
 *       a workspace that is given has at least the size of the widest table's.
 * Supported: head_dim 64 or 128, block_size 16, n_q / n_kv a whole number up
 * to 16, n_kv <= 64, num_seqs <= 4096, max_q_len <= 1024.
 */
size_t vmps_paged_tree_attention_workspace_bytes(int num_seqs, int max_q_len, int n_q, int n_kv,
                                                 int head_dim, int max_blocks_per_seq, int dtype);
int vmps_paged_tree_attention(void* out, const void* q, int64_t q_row_stride, const void* pool,
                              const int32_t* block_tables, int max_blocks_per_seq,
                              const int32_t* ctx_lens, const int32_t* seq_lens,
                              const int32_t* q_lens, const int32_t* cu_q,
                              const int32_t* tree_mask, int mask_words, int num_seqs,
                              int total_q, int max_q_len, int n_q, int n_kv, int head_dim,
                              int block_size, int num_blocks, float scale, void* workspace,
                              size_t workspace_bytes, int dtype, void* stream);

/*
 * Commit of the drafted branch that the model agrees with.  No counterpart
 * in the reference.
 *
 * Sequence i's n = seq_lens[i] - ctx_lens[i] drafted nodes are rows
 * cu_tree[i] .. of parents, tokens and target_ids.  Node 0 is the root (the
 * last token already decided, accepted by definition); parents[node] is the
 * index of an earlier node of the same tree (node 0's is not read).
 * target_ids[node] is the model's own next token after that node.  From the
 * root the walk goes to the lowest-numbered child whose token is
 * target_ids[current] and stops where there is none:
 *   path[i][k]    k-th accepted node, -1 from count[i] on   int32 [num_seqs][max_tree]
 *   count[i]      accepted nodes (0 only if n is 0)         int32 [num_seqs]
 *   next_token[i] target_ids of the last one, -1 if none    int64 [num_seqs]
 * and in every layer of pool ([num_layers][num_blocks][2][16][n_kv][head_dim]
 * contiguous) the K and V of slot ctx + path[k] move to slot ctx + k.  Blocks
 * must not be shared between sequences from slot ctx on.  What the slots past
 * ctx + count hold afterwards is not meaningful.
 * A tree above max_tree (<= 1024) or outside [0, total_nodes) sets error bit
 * 64 and counts as empty; a slot outside the block table or the pool sets bit
 * 4 or 2 and is not moved.  n_kv * head_dim: a multiple of 8, at most 65536.
 */
int vmps_commit_tree(int32_t* path, int32_t* count, int64_t* next_token, void* pool,
                     int num_layers, const int32_t* block_tables, int max_blocks_per_seq,
                     const int32_t* ctx_lens, const int32_t* seq_lens, const int32_t* cu_tree,
                     const int32_t* parents, const int32_t* tokens, const int64_t* target_ids,
                     int num_seqs, int total_nodes, int max_tree, int n_kv, int head_dim,
                     int block_size, int num_blocks, int dtype, void* stream);

/*
 * Products with 4-bit weights (a drafter's projections).  No counterpart in
 * the reference, whose weights are 16-bit nn.Linear modules.
 *   out[m][n] = sum_g scales[n][g] * sum_{k in group g} x[m][k] * (code[n][k] - zeros[n][g])
 * codes:  uint8 [N][K / 2], row n's code k in byte k / 2, the even k in the
 *         low four bits.  scales: [N][K / group_size] in x's type.
 * zeros:  uint8 [N][K / group_size], or NULL for 8 everywhere.
 * All contiguous and 16-byte aligned.  Sums and scaling in fp32, one rounding;
 * codes are carried as 1024 + code, whose share of a group's fp32 sum is taken
 * off again: before its rounding an output is within 2^-12 * sum_k |x| * scale
 * of the formula (for zero points up to 15).  fp16 activations that share their
 * sign come near that, random signs stay below a hundredth of it.
 * A row's infinities and NaN give what the formula gives and reach no other row
 * (such a call takes longer).
 * With silu_mul != 0 the weight is the fused [gate; up] of 2N rows and
 * out[m][n] = silu(gate) * up of the unrounded fp32 products.
 * Shapes: M <= 32, any N, group_size 32, 64 or 128, K a multiple of it below
 * 2^31 - 1023, 2N * K / group_size below 2^31; x
 * 16-byte aligned with rows a multiple of 8 elements apart, out rows at least
 * N apart, 2-byte aligned.  vmps_w4_gemm_supported says whether a shape is
 * built (1) or not (0).
 */
int vmps_w4_gemm_supported(int M, int N, int K, int group_size);
int vmps_w4_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                 const void* codes, const void* scales, const void* zeros, int M, int N, int K,
                 int group_size, int silu_mul, int dtype, void* stream);

/*
 * The 8-bit paged cache (VMPS_CACHE_INT8, VMPS_CACHE_E4M3), half the bytes of
 * the 16-bit pool.  No counterpart in the reference.
 *   codes  [num_blocks][2][16][n_kv][head_dim]  int8 or e4m3 (dim 1: 0 = K, 1 = V)
 *   scales [num_blocks][n_kv][2][16]            fp32
 * both contiguous and 16-byte aligned.  The value stored is code * scale of its
 * token, head and kind (scales of a caller's own may be negative).  Written by
 * vmps_norm_rope_and_cache, the scale is the
 * largest magnitude of the token's head_dim values over 127 (int8) or 448
 * (e4m3) and the code the value times that over the largest magnitude, to nearest
 * with ties to even (rotated and normalised values are fp32, and within 2^-21 of a tie
 * may go to either side; the others go where the exact quotient does).  Rows
 * whose largest magnitude is below 2^-100 are stored as zeros with scale 0; a
 * row that holds an infinity or a NaN has scale NaN and reads as NaN.
 */

/*
 * Norms of queries and keys per head, rotation and cache write in one pass
 * (kernel 9), for attention layers that normalise q and k, and for every layer
 * over an 8-bit cache.  No counterpart in the reference, whose layers have
 * neither; the write takes the place of vmps_rope_reshape_and_cache.
 *   y = x * weight / sqrt(mean(x^2) + eps) over a head's head_dim values of q
 *       and k (q_weight, k_weight: [head_dim] of `dtype`; NULL: y = x)
 *   q_out = rope(y of q); K slot <- rope(y of k); V slot <- v
 * rope() is the rotate-half form with the angle positions[i] * inv_freq[j],
 * whose product is exact (vmps_rope_reshape_and_cache rounds it to fp32, as the
 * reference does).  All of it is fp32 and rounded once, to `dtype` or to a code
 * of `cache_format`; heads with values from about 1e18 on overflow the sum of
 * squares.  inv_freq NULL: no rotation (positions may be NULL).
 *
 * q_out, q, k, v: num_rows rows of heads [heads][head_dim], row strides in
 * elements (multiples of 8, at least a row); q_out may be q where the strides
 * agree, and overlaps neither q otherwise, nor k or v.  n_q 0: keys and values alone.  slot_mapping int32[num_rows]: block *
 * 16 + slot, negative: nothing is cached for the row.  Two rows of a call must
 * not share a slot.  A negative position sets error bit 16 and skips the row, a
 * slot outside the cache sets bit 1 and is not written.  scales: NULL for
 * VMPS_CACHE_16BIT.  Supported: head_dim 64 or 128, block_size 16; all pointers
 * 16-byte aligned.
 */
int vmps_norm_rope_and_cache(void* q_out, int64_t q_out_row_stride, const void* q,
                             int64_t q_row_stride, const void* k, int64_t k_row_stride,
                             const void* v, int64_t v_row_stride, const void* q_weight,
                             const void* k_weight, float eps, const int32_t* positions,
                             const int32_t* slot_mapping, const float* inv_freq, void* cache,
                             float* scales, int num_rows, int n_q, int n_kv, int head_dim,
                             int block_size, int num_blocks, int cache_format, int dtype,
                             void* stream);

/*
 * Pages of the 8-bit cache read back into 16-bit pages (kernel 10), e.g. for
 * vmps_paged_prefill_attention or vmps_paged_tree_attention.  Page j of sequence
 * i, block_tables[i][j], goes to block dst_tables[i][j] of `pool`
 * ([pool_blocks][2][16][n_kv][head_dim] of `dtype`) for j < ceil(seq_lens[i] /
 * 16); both tables have max_blocks_per_seq columns.  Slots at and past
 * seq_lens[i] of the last page are set to zero, other blocks are left as they
 * were.  code * scale is fp32, rounded once.  Two pages must not go to one
 * block.  seq_lens[i] beyond the table sets error bit 4 (the table's pages are
 * read); a block outside the cache or the pool sets bit 2 and is skipped.
 * num_seqs <= 4096, n_kv <= 64, head_dim 64 or 128, block_size 16.
 */
int vmps_read_cache8(void* pool, int pool_blocks, const int32_t* dst_tables, const void* codes,
                     const float* scales, const int32_t* block_tables, int max_blocks_per_seq,
                     const int32_t* seq_lens, int num_seqs, int n_kv, int head_dim,
                     int block_size, int num_blocks, int cache_format, int dtype, void* stream);

/*
 * Decode attention over the 8-bit cache (kernel 11): vmps_paged_decode_attention
 * with K and V read from codes and scales.
 *   out[i][h] = softmax_t(scale * q[i][h] . K[t][h / G]) . V[t][h / G], t < seq_lens[i]
 * Scores, maxima and sums are fp32; for its products with V's codes a softmax weight
 * times V's scale is kept to 2^-22 of itself for fp16 outputs, and rounded to fp16 (2^-11)
 * for bf16 ones, or by 2^-35 of the head's largest such product where that is more (by 2^-17
 * where all of V is about 2^-100).  Weights are counted down to 2^-44 of the largest where V
 * is below 2^100, to 2^-16 at fp32's largest.  q is [num_seqs][n_q][head_dim] with a row
 * stride (a multiple of 8 elements), out contiguous, both 16-byte aligned.  A
 * sequence of length 0 gets a zero row; slots at and past seq_lens[i] take no
 * part, whatever they hold.  seq_lens[i] beyond the table sets error bit 4 (the
 * table's pages are read); a block outside the cache sets bit 2.
 * Supported: head_dim 64 or 128, block_size 16, n_q / n_kv a whole number up to
 * 16, n_kv <= 64, num_seqs <= 4096, num_seqs * (max_blocks_per_seq + 2) below 2^29.
 *
 * The workspace (256-byte aligned) holds the partial results of sequences cut
 * between CTAs and their arrival counters; its size does not depend on the
 * lengths.  Its first 1 MiB (the counters) must be zero before the first call
 * (vmps_paged_decode_workspace_init); every call leaves it zero, so one
 * workspace serves calls of any shape, and vmps_paged_decode_attention's too.
 * Calls that may overlap on the GPU need different workspaces; after error bit
 * 8, when the calls that used it have ended, it is to be zeroed again.  out must not overlap q.  0 bytes: the shape
 * is not supported.
 */
size_t vmps_paged_decode_cache8_workspace_bytes(int num_seqs, int n_q, int n_kv, int head_dim);
int vmps_paged_decode_attention_cache8(void* out, const void* q, int64_t q_row_stride,
                                       const void* codes, const float* scales,
                                       const int32_t* block_tables, int max_blocks_per_seq,
                                       const int32_t* seq_lens, int num_seqs, int n_q, int n_kv,
                                       int head_dim, int block_size, int num_blocks, float scale,
                                       void* workspace, size_t workspace_bytes, int cache_format,
                                       int dtype, void* stream);

/*
 * The three calls above with their arguments in a struct, field by field under the
 * same names, for hosts whose foreign calls cost by the argument (0.2 us each from
 * Python's ctypes, 4 us of 20 for the longest).  The struct is read before the
 * call returns.
 */
typedef struct vmps_norm_rope_args {
  void* q_out;
  const void *q, *k, *v;
  int64_t q_out_row_stride, q_row_stride, k_row_stride, v_row_stride;
  const void *q_weight, *k_weight;
  const int32_t *positions, *slot_mapping;
  const float* inv_freq;
  void* cache;
  float* scales;
  float eps;
  int num_rows, n_q, n_kv, head_dim, block_size, num_blocks, cache_format, dtype;
} vmps_norm_rope_args;
int vmps_norm_rope_and_cache_args(const vmps_norm_rope_args* args, void* stream);

typedef struct vmps_read_args {
  void* pool;
  const int32_t* dst_tables;
  const void* codes;
  const float* scales;
  const int32_t *block_tables, *seq_lens;
  int pool_blocks, max_blocks_per_seq, num_seqs, n_kv, head_dim, block_size, num_blocks,
      cache_format, dtype;
} vmps_read_args;
int vmps_read_cache8_args(const vmps_read_args* args, void* stream);

typedef struct vmps_decode_cache8_args {
  void* out;
  const void* q;
  int64_t q_row_stride;
  const void* codes;
  const float* scales;
  const int32_t *block_tables, *seq_lens;
  void* workspace;
  size_t workspace_bytes;
  float scale;
  int max_blocks_per_seq, num_seqs, n_q, n_kv, head_dim, block_size, num_blocks, cache_format,
      dtype;
} vmps_decode_cache8_args;
int vmps_paged_decode_attention_cache8_args(const vmps_decode_cache8_args* args, void* stream);

/*
 * Copies `bytes` from `src` to `dst` with the GPU's own loads and stores,
 * as a link of a chain of kernels launched with programmatic dependent
 * launch.  No counterpart in the reference (whose inputs never leave host
 * memory).  `src` may be pinned host memory: this is how a serving loop
 * stages a decode step's inputs from the host without a copy-engine copy
 * between two decode steps, which would cost the second step its early
 * launch.  The copy starts while the kernel before it on the stream still
 * runs and does not wait for it; the launch then completes only after that
 * kernel has, so the kernel after it finds both finished.  Therefore `dst`
 * must not be read or written by the kernel immediately before this one on
 * the stream (earlier kernels have completed).  A fused decode step reads
 * its step metadata before its own PDL wait, so between the
 * stage copy of its inputs and the step itself there must be a kernel that
 * waits before it lets the next one start (another decode step): stage
 * step i+1 just before step i (three staging buffers), and stage the first
 * step of a chain with an ordinary copy.  Both pointers 16-byte aligned,
 * bytes a multiple of 16.
 */
int vmps_stage_copy(void* dst, const void* src, size_t bytes, void* stream);

/*
 * Reads and clears the device error word of the current device (a bitwise OR
 * of index violations the kernels skipped since the last call).  Synchronises
 * `stream`.  Bits: 1 slot out of range, 2 block id out of range, 4 seq_len
 * beyond the block table, 8 an internal wait timed out, 16 negative position,
 * 32 a fused-step slot outside the sequence's last page, 64 prefill or tree
 * rows outside [0, total_q) or a q_len (tree) above max_q_len (max_tree).
 */
int vmps_debug_error_word(void* stream, int* word_out);

#ifdef __cplusplus
}
#endif

#endif /* VMPS_H_ */
