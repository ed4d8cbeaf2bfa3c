// Paged attention of drafted tree tokens over a sequence's cache, on the
// sm_100a tensor cores (tcgen05 MMA with TMEM accumulators).
//
// Row r of sequence i (one drafted token, one query head) sees every cached
// slot t < ctx_lens[i] and the drafted slots ctx_lens[i] + j whose bit j is
// set in its mask row:
//     s_t = scale * q . K_t,   out = sum_t e^(s_t - m) V_t / sum_t e^(s_t - m).
// A row that sees no slot is zero.
//
// What bounds it.  Every K and V element is read once for all rows of its kv
// head: 128 rows do 128 flops per byte, so up to about 200 rows per kv head
// the cache stream from HBM is the bound, above that the arithmetic (first
// the softmax, which the MMAs of the other CTA on the SM overlap).  Short calls
// are bound by latency: 3.4 us of plan, 4.5 us to the first scores and, where
// sequences are cut, about 10 us from the last CTA's end to the joined output.
// Measured, 32 query and 8 kv heads of size 128 in bf16, calls in a row: 4 x
// 131072 slots, 16 drafts 332 to 348 us (6.2 to 6.5 TB/s, the copy rate); 32 ragged
// sequences of up to 4096 slots and 26 drafts 78 us (3.7 TB/s); with 64 query
// heads, 8 x 64 drafts over up to 8192 slots 143 to 206 us by the box's power state
// (0.34 to 0.49 of the bf16 peak; the softmax warps spill registers).  One sequence
// of 137 slots (heads 32/4 x 64) takes 9.5 us, and 13.5 where the tables are wide
// enough for contexts that would be cut.
//
// Work split.  A row tile is 128 MMA rows: 128 / G drafted tokens x the G
// query heads of a kv head, so K and V are read once per kv head and GQA is
// never materialised.  Within one row tile index the key tiles (64 keys, 4
// pages) of all sequences and kv heads are laid end to end, each sequence
// start weighing kSegWeight / kTileWeight tiles, and every CTA of a
// persistent grid (2 per SM) takes one contiguous, equal share: ragged
// batches and a few long contexts both fill the machine.  Row tile indices
// get CTAs in proportion to their work, each starting on a CTA of its own, so
// that the row tiles of one context stream the same pages at the same time
// (the second reader finds them in L2).  Every CTA works the plan out from the
// lengths on the device; the host needs none of them.
//
// A sequence cut between CTAs: each piece stores its running maximum, sum and
// unnormalised output in fp32, and a second small kernel (programmatic
// dependent launch) joins the pieces in a fixed order.  Calls whose block
// tables are at most kWholeTiles key tiles wide are never cut and skip it.
//
// Data movement, MMA order and softmax are those of the prefill kernel (warp 4
// loads Q and K pages, warp 5 V pages, warp 6 issues the MMAs, warps 0-3 own a
// row per thread; S is double-buffered in TMEM, P overwrites S and is PV's A
// operand), run as one pipeline over all tiles of all segments of the CTA's
// share: the next segment's first tiles load and multiply while the current
// one finishes.
//
// Masks.  Tiles inside the cached context need none.  In a tile that reaches
// past it a row's 64 visibility bits are cut out of its mask words; masked
// scores become -inf before the maximum.  There V is also cleaned in shared
// memory: rows past the sequence's end are zeroed and non-finite values of
// drafted tokens are replaced by 0 (0 * inf would reach rows that do not see
// them); a row that does see such a value adds it in its epilogue.
//
// Rounding: P is rounded to the 16-bit type as PV's operand (its sum is not),
// the output once; scores, maxima, sums and accumulators are fp32.  fp16 has no
// bits to spare below 2^-14, so its P is 2^kLift times as large: weights down to
// 2^-21 of the row's largest keep all their bits, and what one loses below that is
// at most 2^-32 of the largest (2^-25 without: many small weights behind a large
// one then vanish from the product while the sum they are divided by has them).
//
// Safety.  Every mbarrier wait is bounded; a wait that gives up sets
// kDevErrTimeout and a CTA-wide abort flag, the loads and MMAs stop being
// issued, those in flight are waited for (bounded) and the TMEM is always freed.
#include <mutex>

#include "tree_plan.h"
#include "vmps_abi_internal.h"
#include "vmps_common.cuh"
#include "vmps_tcgen05.cuh"

namespace vmps {
namespace {

constexpr int kPage = 16;
constexpr int kTtRows = 128;                  // MMA M
constexpr int kTtPages = kTtKeys / kPage;
constexpr int kTtThreads = 224;
constexpr int kTtKWarp = 4, kTtVWarp = 5, kTtMmaWarp = 6;
constexpr int kTtQChunk = kTtRows * 128;      // 128 rows x 64 16-bit columns
constexpr int kTtKChunk = kTtKeys * 128;
constexpr int kTtCtasPerSm = 2;
constexpr int kTtMaxSeqs = 4096;
constexpr int kTtMaxQLen = 1024;
constexpr int kTtMaxRowTiles = 128;           // 1024 tokens x 16 heads / 128
// The running maximum bounds a score to within 2^kSlack; P <= 2^(kSlack + kLift),
// which is below fp16's 65504.
constexpr float kSlack = 8.f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int kMergeThreads = 256;
constexpr int kMergeBlocksPerSm = 2;
constexpr int kMergeCols = 16;                // output columns per merge unit
constexpr int kMaxCtas = 512;

template <int D>
struct TreeShape {
  // K ring and V ring depth: what fits beside Q with two CTAs on an SM.
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kChunks = D / 64;
  static constexpr int kQBytes = kChunks * kTtQChunk;
  static constexpr int kTileBytes = kChunks * kTtKChunk;  // K (or V) of one key tile
  static constexpr int kBarBytes = 512 + kTtMaxRowTiles * 4;
  static constexpr int kFixedBytes = kQBytes + 2 * kStages * kTileBytes + kBarBytes;
  static constexpr uint32_t kTmemCols = 256;  // S 2 x 64 columns, O up to 128
};

struct TreeParams {
  void* out;
  const void* pool;
  const int32_t* block_tables;
  const int32_t* ctx_lens;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  const int32_t* cu_q;
  const uint32_t* mask;
  int mask_words, max_blocks, num_seqs, total_q, max_q_len, n_q, n_kv, G, num_blocks;
  int tokens_per_tile, row_tiles, n_cta, whole, box_tokens;
  int part_rows;     // rows of a partial record (a multiple of 32)
  float scale_log2;
  int* records;      // [6][n_cta]: the cut sequence whose second piece CTA b holds, -1 if none
  float2* part_ml;   // [n_cta * 2][part_rows]
  float4* part_o;    // [n_cta * 2][D / 4][part_rows]
  int* err;
};

struct TreeSeq {
  int ctx, n, q_len, row0;
};

// Lengths of a sequence, clamped to what the buffers hold.
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int s, bool report) {
  TreeSeq r;
  r.n = p.seq_lens[s];
  r.ctx = p.ctx_lens[s];
  r.q_len = p.q_lens[s];
  r.row0 = p.cu_q[s];
  if (r.q_len <= 0) {
    r.q_len = 0;
  } else if (r.row0 < 0 || static_cast<long long>(r.row0) + r.q_len > p.total_q) {
    if (report) set_error(p.err, kDevErrQueryRange);
    r.q_len = 0;
  } else if (r.q_len > p.max_q_len) {
    if (report) set_error(p.err, kDevErrQueryRange);
    r.q_len = p.max_q_len;
  }
  if (r.n > p.max_blocks * kPage) {
    if (report) set_error(p.err, kDevErrSeqLen);
    r.n = p.max_blocks * kPage;
  }
  if (r.n < 0) r.n = 0;
  r.ctx = min(max(r.ctx, 0), r.n);
  return r;
}

// 64 visibility bits of a row for keys [t0, t0 + 64).
__device__ __forceinline__ uint64_t tree_visible(const uint32_t* mrow, int words, int t0, int ctx,
                                                 int n) {
  const int lead = ctx - t0;  // keys below this are cached context
  uint64_t vis = lead >= 64 ? ~0ull : (lead > 0 ? (1ull << lead) - 1 : 0ull);
  if (lead < 64) {
    const int sh = lead > 0 ? lead : 0;
    const int bit = lead > 0 ? 0 : -lead;  // first draft of the tile
    const int w = bit >> 5;
    const uint32_t w0 = w < words ? mrow[w] : 0u;
    const uint32_t w1 = w + 1 < words ? mrow[w + 1] : 0u;
    const uint32_t w2 = w + 2 < words ? mrow[w + 2] : 0u;
    const uint32_t lo = __funnelshift_r(w0, w1, bit & 31);
    const uint32_t hi = __funnelshift_r(w1, w2, bit & 31);
    vis |= ((static_cast<uint64_t>(hi) << 32) | lo) << sh;
  }
  const int left = n - t0;
  if (left < 64) vis &= left > 0 ? (1ull << left) - 1 : 0ull;
  return vis;
}

// Whether either 16-bit half is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool nonfinite16(uint32_t half) {
  const uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (half & e) == e;
}

// Sum of the non-finite values that the drafts t_begin .. t_end - 1 which a row
// sees hold in column d: they were kept out of the MMA.  Only ever runs after
// such a value was found.
template <typename T, int D>
__device__ __noinline__ float tree_nonfinite(const TreeParams& p, const uint32_t* mrow, int s,
                                             int kvh, int ctx, int t_begin, int t_end, int d) {
  float sum = 0.f;
  for (int t = max(t_begin, ctx); t < t_end; ++t) {
    const int j = t - ctx;
    if ((j >> 5) >= p.mask_words || !((mrow[j >> 5] >> (j & 31)) & 1u)) continue;
    const int b = p.block_tables[static_cast<size_t>(s) * p.max_blocks + t / kPage];
    if (b < 0 || b >= p.num_blocks) continue;
    const float x = Elt<T>::to_f(static_cast<const T*>(
        p.pool)[(((static_cast<int64_t>(b) * 2 + 1) * kPage + t % kPage) * p.n_kv + kvh) * D + d]);
    if (!(fabsf(x) <= 3.4e38f)) sum += x;
  }
  return sum;
}

// Waits for a phase; false once a wait has given up (this one or another's:
// the CTA's abort flag), which only the slow path looks at.
__device__ __forceinline__ bool tt_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitLimitCycles) {
      set_error(err, kDevErrTimeout);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void tt_pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void tt_pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Orders this thread's shared-memory writes before later reads by the async
// proxy (MMA operands).
__device__ __forceinline__ void tt_fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kTtThreads, kTtCtasPerSm)
    paged_tree_kernel(const __grid_constant__ CUtensorMap kv_map,
                      const __grid_constant__ CUtensorMap q_map,
                      const __grid_constant__ TreeParams p) {
  using Shape = TreeShape<D>;
  constexpr int KEYS = kTtKeys;
  // The swizzled tiles need 1024-byte alignment; the dynamic window is
  // declared so, and a launch that did not get it reports it and does nothing.
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) set_error(p.err, kDevErrTimeout);
    return;
  }
  uint8_t* sQ = smem_raw;
  uint8_t* sK = sQ + Shape::kQBytes;
  uint8_t* sV = sK + Shape::kStages * Shape::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + Shape::kStages * Shape::kTileBytes);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;  // the segment's last QK is done with Q
  // [2]: MMA -> softmax, PV of a tile complete, by tile parity.  S of tile i in
  // TMEM says that PV(i - 2) has completed but not PV(i - 1): with one barrier
  // the parity of PV(i) could be taken for PV(i - 2)'s.
  uint64_t* o_ready = bars + 2;
  uint64_t* s_full = bars + 4;   // [2]: S in TMEM buffer (tile & 1)
  uint64_t* p_full = bars + 6;   // [2]: softmax -> MMA, P in that buffer and O rescaled
  uint64_t* mma_done = bars + 8; // everything issued has completed
  uint64_t* k_full = bars + 9;
  uint64_t* k_empty = k_full + Shape::kStages;
  uint64_t* v_full = k_empty + Shape::kStages;
  uint64_t* v_empty = v_full + Shape::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + Shape::kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // Segment number (+1) whose V held a non-finite draft, by segment modulo 4.
  // Two entries are not enough: a warp without rows of its own cleans V and
  // skips the epilogues, and can be two segments ahead of one that has yet to
  // read its entry (S(i + 2) follows PV(i), whatever the epilogue of the segment
  // that ends with tile i does).  It is never three ahead: S(i + 3) follows
  // PV(i + 1), for which every warp must have arrived in the segment after.
  volatile int* odd_seg = abort_flag + 1;  // [4]
  TreeShare* share = reinterpret_cast<TreeShare*>(smem_raw + (reinterpret_cast<uint8_t*>(bars) - smem_raw) + 256);
  int* rt_weight = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* wpref = rt_weight + kTtMaxRowTiles;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_seqs = p.num_seqs;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(mma_done, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(o_ready + b, 1);
      mbar_init(s_full + b, 1);
      mbar_init(p_full + b, 4);
    }
    for (int st = 0; st < Shape::kStages; ++st) {
      mbar_init(k_full + st, 1);
      mbar_init(k_empty + st, 1);
      mbar_init(v_full + st, 1);
      mbar_init(v_empty + st, 1);
    }
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) odd_seg[i] = 0;
    fence_mbar_init();
  }
  if (warp == kTtMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(Shape::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (p.box_tokens * p.G < kTtRows) {
    // Rows the Q loads never write: zeros, so their scores raise no maximum.
    for (int i = threadIdx.x; i < Shape::kQBytes / 16; i += kTtThreads) {
      reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    tt_fence_async();
  }
  if (lane == 0 && warp == kTtKWarp) prefetch_tmap(&q_map);
  if (lane == 0 && warp == kTtVWarp) prefetch_tmap(&kv_map);
  tt_pdl_wait();  // the lengths, q and the pool may come from the kernel before
  tt_pdl_trigger();

  // ── plan ───────────────────────────────────────────────────────────────────
  // wpref[s + 1] first holds sequence s's tiles (upper bits) and how many row
  // tiles it has (lower 8), so that the lengths are read from memory once.
  for (int s = threadIdx.x; s < num_seqs; s += kTtThreads) {
    const TreeSeq q = tree_seq(p, s, blockIdx.x == 0);
    wpref[s + 1] = (tree_tiles(q.n) << 8) | ((q.q_len + p.tokens_per_tile - 1) / p.tokens_per_tile);
  }
  __syncthreads();
  for (int rt = warp; rt < p.row_tiles; rt += kTtThreads / 32) {
    int sum = 0;
    for (int s = lane; s < num_seqs; s += 32) sum += tree_weight(wpref[s + 1], rt);
    for (int sh = 16; sh; sh >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
    if (lane == 0) rt_weight[rt] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    // Every lane does the same (the divisions are what takes the time).
    long long total = 0;
    int used = 0;  // row tile indices with work: the first ones
    for (int rt = 0; rt < p.row_tiles && rt_weight[rt] > 0; ++rt, ++used) {
      total += static_cast<long long>(rt_weight[rt]) * p.n_kv;
    }
    const long long chunk = tree_chunk(total, used, p.n_cta, p.whole);
    int first = 0, rt = 0;
    for (; rt < used; ++rt) {
      const long long w = static_cast<long long>(rt_weight[rt]) * p.n_kv;
      const int n = static_cast<int>(tree_div(w + chunk - 1, chunk));
      if (static_cast<int>(blockIdx.x) < first + n) break;
      first += n;
    }
    if (rt == used) rt = -1;
    int carry = 0;
    for (int base = 0; base < num_seqs; base += 32) {
      const int s = base + lane;
      int v = rt >= 0 && s < num_seqs ? tree_weight(wpref[s + 1], rt) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      if (s < num_seqs) wpref[s + 1] = v + carry;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) wpref[0] = 0;
    __syncwarp();
    // Lane 0 finds the share's begin, lane 1 its end.
    if (lane < 2) {
      TreePos b;
      b.kvh = b.s = b.j = 0;
      if (rt >= 0) {
        const long long w0 = static_cast<long long>(blockIdx.x - first + lane) * chunk;
        b = tree_pos(wpref, num_seqs, p.n_kv, p.whole, w0);
      }
      if (lane == 0) {
        share->rt = rt;
        share->first_cta = first;
        share->chunk = chunk;
        share->begin = b;
      } else {
        share->end = b;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const TreeShare& sh = *share;
  // Up to 64 rows need the softmax of two warps (or one).  The two CTAs of an SM
  // then use different ones -- they hold different halves of its TMEM -- so
  // that their exponentials do not queue for the same quarter of the SM.
  const int row_shift = p.box_tokens * p.G <= kTtRows / 2 ? ((tmem_base >> 8) & 1) * (kTtRows / 2) : 0;
  const int tok0 = sh.rt * p.tokens_per_tile;

  if (warp == kTtKWarp || warp == kTtVWarp) {
    // ── loads: one warp streams K tiles (and Q), another V tiles ──────────────
    const bool is_v = warp == kTtVWarp;
    const int oob = 2 * p.num_blocks;  // past the pool: the TMA fills zeros
    uint64_t* full = is_v ? v_full : k_full;
    // With two ring slots the slot and the tile parity are one, and the barrier
    // that tells the softmax of a product tells the loader of its free slot.
    uint64_t* empty = Shape::kStages == 2 ? (is_v ? o_ready : s_full) : (is_v ? v_empty : k_empty);
    uint8_t* ring = is_v ? sV : sK;
    auto fetch = [&](int s, int n_pages, int page) -> int {  // block id of `page`, or -1
      if (page >= n_pages) return -1;
      const int b = p.block_tables[static_cast<size_t>(s) * p.max_blocks + page];
      if (b < 0 || b >= p.num_blocks) {
        set_error(p.err, kDevErrBlockRange);
        return -1;
      }
      return b;
    };
    TreeWalk w;
    w.start(wpref, num_seqs, sh);
    int it = 0, seg = 0;
    bool go = true;
    int first_ids = -1;  // this lane's page of the segment's first 32
    TreeSeq q = {};
    if (w.valid) {
      q = tree_seq(p, w.at.s, false);
      first_ids = fetch(w.at.s, (q.n + kPage - 1) / kPage, w.at.j * kTtPages + lane);
    }
    while (w.valid && go) {
      const int s = w.at.s, kvh = w.at.kvh, j0 = w.at.j, j1 = w.j1;
      const int n_pages = (q.n + kPage - 1) / kPage;
      const int page_begin = j0 * kTtPages;
      int ids = first_ids;
      int nxt = fetch(s, n_pages, page_begin + 32 + lane);
      if (!is_v && lane == 0) {
        if (seg > 0 && !tt_wait(q_empty, (seg - 1) & 1, abort_flag, p.err)) {
          go = false;
        } else {
          mbar_arrive_expect_tx(q_full, Shape::kChunks * p.box_tokens * p.G * 128);
#pragma unroll
          for (int c = 0; c < Shape::kChunks; ++c) {
            tma_load_3d(sQ + c * kTtQChunk + row_shift * 128, &q_map, q_full, c * 64, kvh * p.G, q.row0 + tok0);
          }
        }
      }
      go = __shfl_sync(0xffffffffu, go ? 1 : 0, 0);
      if (!go) break;
      ++seg;
      // The next segment's lengths and first block ids, long before they are needed.
      w.next(wpref, num_seqs, sh);
      if (w.valid) {
        q = tree_seq(p, w.at.s, false);
        first_ids = fetch(w.at.s, (q.n + kPage - 1) / kPage, w.at.j * kTtPages + lane);
      }
      for (int j = j0; j < j1; ++j, ++it) {
        const int page0 = (j - j0) * kTtPages;  // within the segment
        if (page0 > 0 && (page0 & 31) == 0) {
          ids = nxt;
          nxt = fetch(s, n_pages, page_begin + page0 + 32 + lane);
        }
        int blk[kTtPages];
#pragma unroll
        for (int pg = 0; pg < kTtPages; ++pg) {
          blk[pg] = __shfl_sync(0xffffffffu, ids, (page0 + pg) & 31);
        }
        if (lane == 0) {
          const int st = it % Shape::kStages;
          if (it >= Shape::kStages &&
              !tt_wait(empty + st, ((it / Shape::kStages) - 1) & 1, abort_flag, p.err)) {
            go = false;
          } else {
            mbar_arrive_expect_tx(full + st, Shape::kTileBytes);
#pragma unroll
            for (int pg = 0; pg < kTtPages; ++pg) {
              const int coord = blk[pg] < 0 ? oob : 2 * blk[pg] + (is_v ? 1 : 0);
#pragma unroll
              for (int c = 0; c < Shape::kChunks; ++c) {
                tma_load_4d(ring + st * Shape::kTileBytes + c * kTtKChunk + pg * 2048, &kv_map,
                            full + st, c * 64, 0, kvh, coord);
              }
            }
          }
        }
        go = __shfl_sync(0xffffffffu, go ? 1 : 0, 0);
        if (!go) break;
      }
    }
    // Whatever happened, this warp's own loads land before the shared memory
    // is released.
    if (lane == 0) {
      if (!is_v && seg > 0) mbar_wait(q_full, (seg - 1) & 1, p.err);
      for (int i = max(0, it - Shape::kStages); i < it; ++i) {
        mbar_wait(full + (i % Shape::kStages), (i / Shape::kStages) & 1, p.err);
      }
    }
  } else if (warp == kTtMmaWarp) {
    // ── MMA issue: QK(0), QK(1), then per tile i: PV(i) after its softmax,
    // QK(i + 2) into the S buffer PV(i) just read P from (the MMAs of one
    // thread execute in issue order).  Tiles are numbered through all segments.
    if (lane == 0) {
      const uint32_t t_o = tmem_base + 2 * KEYS;
      const uint32_t idesc_qk = f16_idesc<T>(KEYS, false);
      const uint32_t idesc_pv = f16_idesc<T>(D, true);
      // One lane issues everything, so what it does per MMA counts: operand
      // descriptors are a base (one per ring slot) plus a constant.
      const uint64_t q_desc = sw128_desc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sw128_desc(smem_u32(sK), 16, 1024);
      const uint64_t v_desc = sw128_desc(smem_u32(sV), kTtKChunk, 1024);
      constexpr uint64_t kTileStep = Shape::kTileBytes >> 4;
      TreeWalk wq, wp;  // the next QK's segment, the next PV's segment
      wq.start(wpref, num_seqs, sh);
      wp = wq;
      int left_q = wq.valid ? wq.j1 - wq.at.j : 0, left_p = left_q;
      int seg_q = 0, iq = 0, ip = 0;
      bool new_q = true, first = true;
      auto issue_qk = [&]() -> bool {  // one tile, if any is left
        if (!wq.valid) return true;
        const int st = iq % Shape::kStages;
        if (new_q && !tt_wait(q_full, seg_q & 1, abort_flag, p.err)) return false;
        if (!tt_wait(k_full + st, (iq / Shape::kStages) & 1, abort_flag, p.err)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + st * kTileStep;
        const uint32_t t_s = tmem_base + (iq & 1) * KEYS;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          tc_mma(t_s, q_desc + (((k >> 2) * kTtQChunk + (k & 3) * 32) >> 4),
                 kd + (((k >> 2) * kTtKChunk + (k & 3) * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u);
        }
        if (Shape::kStages != 2) tc_commit(k_empty + st);
        tc_commit(s_full + (iq & 1));
        ++iq;
        new_q = false;
        if (--left_q == 0) {
          tc_commit(q_empty);
          wq.next(wpref, num_seqs, sh);
          left_q = wq.j1 - wq.at.j;
          new_q = true;
          ++seg_q;
        }
        return true;
      };
      bool ok = issue_qk() && issue_qk();
      while (ok && wp.valid) {
        const int st = ip % Shape::kStages;
        if (!tt_wait(v_full + st, (ip / Shape::kStages) & 1, abort_flag, p.err) ||
            !tt_wait(p_full + (ip & 1), (ip >> 1) & 1, abort_flag, p.err)) {
          break;
        }
        tc_fence_after();
        const uint64_t vd = v_desc + st * kTileStep;
        const uint32_t t_p = tmem_base + (ip & 1) * KEYS;
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k) {
          // A segment's first PV overwrites O.
          tc_mma_ts(t_o, t_p + k * 8, vd + ((k * 2048) >> 4), idesc_pv, (!first || k > 0) ? 1u : 0u);
        }
        if (Shape::kStages != 2) tc_commit(v_empty + st);
        tc_commit(o_ready + (ip & 1));
        ++ip;
        first = false;
        if (--left_p == 0) {
          wp.next(wpref, num_seqs, sh);
          left_p = wp.j1 - wp.at.j;
          first = true;
        }
        ok = issue_qk();
      }
      // Every MMA this lane issued completes before the TMEM is freed.
      tc_commit(mma_done);
      mbar_wait(mma_done, 0, p.err);
    }
  } else {
    // ── softmax and epilogue: one row per thread ─────────────────────────────
    const int m = threadIdx.x - row_shift;  // row; TMEM lane threadIdx.x
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t t_o = tmem_base + lane_base + 2 * KEYS;
    const int t_row = max(m, 0) / p.G;  // drafted token of the row tile
    const int head_in_group = m - t_row * p.G;
    const float scale = p.scale_log2;
    // (After a wait that gave up these warps go through the motions on whatever
    // TMEM holds: nothing they touch is anyone else's.)
    int it = 0, seg = 0;
    if (threadIdx.x == 0 && !p.whole) p.records[blockIdx.x] = -1;
    TreeWalk w;
    w.start(wpref, num_seqs, sh);
    while (w.valid) {
      const int s = w.at.s, kvh = w.at.kvh, j0 = w.at.j, j1 = w.j1, tiles = w.tiles;
      const TreeSeq q = tree_seq(p, s, false);
      const int rows = min(p.tokens_per_tile, q.q_len - tok0) * p.G;
      const bool active = warp * 32 >= row_shift && warp * 32 - row_shift < rows;  // warp-uniform
      const bool valid = m >= 0 && m < rows;
      const int row = q.row0 + tok0 + (valid ? t_row : 0);
      const uint32_t* mrow = p.mask + static_cast<size_t>(row) * p.mask_words;
      float m_run = -INFINITY;
      float l_run = 0.f;
      for (int j = j0; j < j1; ++j, ++it) {
        tt_wait(s_full + (it & 1), (it >> 1) & 1, abort_flag, p.err);
        __syncwarp();
        const int key0 = j * KEYS;
        const bool tail = key0 + KEYS > q.ctx;  // reaches drafts or the end
        if (tail) {
          // Clean V: every warp takes its share of the tile's 128-byte lines.
          const int st = it % Shape::kStages;
          tt_wait(v_full + st, (it / Shape::kStages) & 1, abort_flag, p.err);
          if (threadIdx.x < Shape::kChunks * KEYS) {
            const int t = key0 + (threadIdx.x & (KEYS - 1));
            uint4* line = reinterpret_cast<uint4*>(sV + st * Shape::kTileBytes + threadIdx.x * 128);
            if (t >= q.n) {
#pragma unroll
              for (int u = 0; u < 8; ++u) line[u ^ (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
            } else if (t >= q.ctx) {
              bool found = false;
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                uint4 x = line[u ^ (lane & 7)];
                uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if (nonfinite16<T>(xs[i] & 0xffffu)) { xs[i] &= 0xffff0000u; odd = true; }
                  if (nonfinite16<T>(xs[i] >> 16)) { xs[i] &= 0x0000ffffu; odd = true; }
                }
                if (odd) {
                  line[u ^ (lane & 7)] = x;
                  found = true;
                }
              }
              if (found) odd_seg[seg & 3] = seg + 1;
            }
          }
          tt_fence_async();
        }
        if (active) {
          tc_fence_after();
          const uint32_t t_s = tmem_base + lane_base + (it & 1) * KEYS;
          uint32_t sc[KEYS / 16][16];
#pragma unroll
          for (int c = 0; c < KEYS / 16; ++c) tmem_ld16(t_s + c * 16, sc[c]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < KEYS / 16; ++c) tmem_ld_fence_regs(sc[c]);
          if (tail) {
            const uint64_t vis = valid ? tree_visible(mrow, p.mask_words, key0, q.ctx, q.n) : 0ull;
            const uint32_t v0 = static_cast<uint32_t>(vis), v1 = static_cast<uint32_t>(vis >> 32);
#pragma unroll
            for (int c = 0; c < KEYS / 16; ++c) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int bit = (c & 1) * 16 + i;
                if (!(((c < 2 ? v0 : v1) >> bit) & 1u)) sc[c][i] = __float_as_uint(-INFINITY);
              }
            }
          }
          // The maximum is taken on raw scores (the scale is positive) in four
          // independent chains; the scale is folded into the exponent.
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < KEYS / 16; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              mx4[i & 3] = fmax3(mx4[i & 3], __uint_as_float(sc[c][2 * i]),
                                 __uint_as_float(sc[c][2 * i + 1]));
            }
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale;
          const float m_new = fmaxf(m_run, mx);
          if (j == j0) {
            m_run = m_new;
          } else if (__any_sync(0xffffffffu, m_new > m_run + kSlack)) {
            // The running maximum only has to bound the scores to within 2^kSlack:
            // O is rescaled (once the PV before has landed) when it grew by more.
            tt_wait(o_ready + ((it - 1) & 1), ((it - 1) >> 1) & 1, abort_flag, p.err);
            __syncwarp();
            tc_fence_after();
            // -inf - -inf: a row that has seen nothing yet keeps its zeros.
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + c * 16, o);
              tmem_ld_wait();
              tmem_ld_fence_regs(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(t_o + c * 16, o);
            }
            l_run *= alpha;
            m_run = m_new;
          }
          uint32_t pk[KEYS / 32][16];
          uint64_t acc2[2] = {0ull, 0ull};
          const float base = m_run == -INFINITY ? 0.f : m_run - kLift<T>;
          const uint64_t scale2 = f2_make(scale, scale);
          const uint64_t neg_m2 = f2_make(-base, -base);
#pragma unroll
          for (int c = 0; c < KEYS / 16; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float a, b;
              f2_split(f2_fma(f2_make(__uint_as_float(sc[c][2 * i]),
                                      __uint_as_float(sc[c][2 * i + 1])),
                              scale2, neg_m2),
                       a, b);
              a = fast_exp2(a);
              b = fast_exp2(b);
              acc2[i & 1] = f2_add(acc2[i & 1], f2_make(a, b));
              pk[c >> 1][(c & 1) * 8 + i] = Elt<T>::pack(a, b);
            }
          }
          float s0, s1, s2, s3;
          f2_split(acc2[0], s0, s1);
          f2_split(acc2[1], s2, s3);
#pragma unroll
          for (int c = 0; c < KEYS / 32; ++c) tmem_st16(t_s + c * 16, pk[c]);
          tmem_st_wait();
          l_run += (s0 + s1) + (s2 + s3);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + (it & 1));
      }
      // ── the segment's result ──────────────────────────────────────────────
      const bool complete = j0 == 0 && j1 == tiles;
      int slot = 0;
      if (!complete) {
        const int c0 = tree_owner(wpref, num_seqs, sh, kvh, s, 0) + sh.first_cta;
        slot = c0 == static_cast<int>(blockIdx.x) ? 1 : 0;
        if (c0 + 1 == static_cast<int>(blockIdx.x) && threadIdx.x == 0) {
          // The sequence began in the CTA before this one: this CTA describes
          // the join of its pieces (it has the second of them).
          int* rec = p.records + blockIdx.x;
          rec[0] = s;
          rec[p.n_cta] = kvh;
          rec[2 * p.n_cta] = tok0;
          rec[3 * p.n_cta] = c0;
          rec[4 * p.n_cta] = tree_owner(wpref, num_seqs, sh, kvh, s, tiles - 1) + sh.first_cta;
          rec[5 * p.n_cta] = rows;
        }
      }
      if (active) {
        tt_wait(o_ready + ((it - 1) & 1), ((it - 1) >> 1) & 1, abort_flag, p.err);
        __syncwarp();
        tc_fence_after();
        const bool odd = odd_seg[seg & 3] == seg + 1;
        // A row that saw nothing has l = 0 and O = 0.
        const float inv_l = l_run == 0.f ? 0.f : 1.f / l_run;
        const size_t piece = static_cast<size_t>(blockIdx.x) * 2 + slot;
        T* orow = static_cast<T*>(p.out) +
                  (static_cast<size_t>(row) * p.n_q + kvh * p.G + head_in_group) * D;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(t_o + c * 16, o);
          tmem_ld_wait();
          tmem_ld_fence_regs(o);
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(o[i]);
          if (odd && valid) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              f[i] += tree_nonfinite<T, D>(p, mrow, s, kvh, q.ctx, j0 * KEYS, min(j1 * KEYS, q.n),
                                           c * 16 + i);
            }
          }
          if (complete) {
            uint32_t packed[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) packed[i] = Elt<T>::pack(f[2 * i] * inv_l, f[2 * i + 1] * inv_l);
            if (valid) {
              uint4* dst = reinterpret_cast<uint4*>(orow + c * 16);
              dst[0] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
              dst[1] = make_uint4(packed[4], packed[5], packed[6], packed[7]);
            }
          } else {
            // Column-quad major, so that a warp's 32 rows are adjacent.
            float4* dst = p.part_o + (piece * (D / 4) + c * 4) * p.part_rows + m;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              dst[static_cast<size_t>(i) * p.part_rows] =
                  make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
            }
          }
        }
        if (!complete) p.part_ml[piece * p.part_rows + m] = make_float2(m_run, l_run);
        tc_fence_before();
      }
      ++seg;
      w.next(wpref, num_seqs, sh);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kTtMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(Shape::kTmemCols)
                 : "memory");
  }
}

// Joins the pieces of cut sequences.  A unit is 32 rows x 16 columns of one of
// them.  A unit's pieces go to 1, 2, 4 or 8 warps of a block (as many as the
// number of units leaves idle otherwise: a batch has many sequences of two or
// three pieces, a long context few of dozens), each taking every n-th piece,
// and the warps' results are joined through shared memory, all in a fixed
// order.  Bound: the partial results, read from L2; one warp per unit alone
// took 19 us for 74 pieces of 4 kv heads, eight always 30 us for 256 items of
// two pieces.  The records are brought into shared memory once: read per unit
// they cost 1 us in 79.
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads, kMergeBlocksPerSm)
    paged_tree_merge_kernel(const __grid_constant__ TreeParams p) {
  constexpr int kWarps = kMergeThreads / 32;
  constexpr int kQuads = kMergeCols / 4;
  constexpr int kColUnits = D / kMergeCols;
  constexpr int kBatch = 4;     // pieces in flight per warp
  __shared__ int s_rec[kMaxCtas][6];  // the joins, in order
  __shared__ int s_count[kWarps];
  __shared__ float s_ml[kWarps][32][2];
  __shared__ float4 s_o[kWarps][kQuads][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  tt_pdl_wait();
  constexpr int kRecords = kMaxCtas / kMergeThreads;  // a thread's, loaded together
  int rec[kRecords][6];
  unsigned mask[kRecords];
#pragma unroll
  for (int r = 0; r < kRecords; ++r) {
    const int b = r * kMergeThreads + threadIdx.x;
    rec[r][0] = -1;
    if (b < p.n_cta) {
#pragma unroll
      for (int i = 0; i < 6; ++i) rec[r][i] = p.records[i * p.n_cta + b];
    }
  }
  int n_warp = 0;
#pragma unroll
  for (int r = 0; r < kRecords; ++r) {
    mask[r] = __ballot_sync(0xffffffffu, rec[r][0] >= 0);
    n_warp += __popc(mask[r]);
  }
  if (lane == 0) s_count[warp] = n_warp;
  __syncthreads();
  int at = 0, n_items = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) at += s_count[i];
    n_items += s_count[i];
  }
#pragma unroll
  for (int r = 0; r < kRecords; ++r) {
    if (rec[r][0] >= 0) {
      int* dst = s_rec[at + __popc(mask[r] & ((1u << lane) - 1))];
#pragma unroll
      for (int i = 0; i < 6; ++i) dst[i] = rec[r][i];
    }
    at += __popc(mask[r]);
  }
  __syncthreads();
  const int row_units = p.part_rows / 32;
  const int units = n_items * row_units * kColUnits;
  int per_unit = 1;  // warps
  while (per_unit < kWarps && units * per_unit * 2 <= static_cast<int>(gridDim.x) * kWarps) per_unit *= 2;
  const int groups = kWarps / per_unit;  // units a block works on at once
  const int sub = warp & (per_unit - 1), group = warp / per_unit;
  for (int first = blockIdx.x * groups; first < units; first += gridDim.x * groups) {
    const int unit = first + group;
    const int item = unit / (row_units * kColUnits);
    const int rest = unit - item * (row_units * kColUnits);
    const int ru = rest / kColUnits, cu = rest - ru * kColUnits;
    int s = 0, kvh = 0, tok0 = 0, c0 = 0, c1 = -1, rows = 0;
    if (unit < units) {
      const int* rec = s_rec[item];
      s = rec[0];
      kvh = rec[1];
      tok0 = rec[2];
      c0 = rec[3];
      c1 = rec[4];
      rows = rec[5];
    }
    const bool on = ru * 32 < rows;
    const int row = ru * 32 + lane;
    float m_run = -INFINITY, l_run = 0.f;
    float4 o[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto fold = [&](float m2, float l2, const float4* v) {
      const float mn = fmaxf(m_run, m2);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float a = fast_exp2(m_run - base), b = fast_exp2(m2 - base);
      l_run = l_run * a + l2 * b;
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        o[i].x = o[i].x * a + v[i].x * b;
        o[i].y = o[i].y * a + v[i].y * b;
        o[i].z = o[i].z * a + v[i].z * b;
        o[i].w = o[i].w * a + v[i].w * b;
      }
      m_run = mn;
    };
    if (on) {
      for (int c = c0 + sub; c <= c1; c += per_unit * kBatch) {
        float2 ml[kBatch];
        float4 v[kBatch][kQuads];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int cc = c + k * per_unit;
          if (cc <= c1) {
            const size_t piece = static_cast<size_t>(cc) * 2 + (cc == c0 ? 1 : 0);
            ml[k] = __ldcg(p.part_ml + piece * p.part_rows + row);
            const float4* src = p.part_o + (piece * (D / 4) + cu * kQuads) * p.part_rows + row;
#pragma unroll
            for (int i = 0; i < kQuads; ++i) v[k][i] = __ldcg(src + static_cast<size_t>(i) * p.part_rows);
          }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (c + k * per_unit <= c1) fold(ml[k].x, ml[k].y, v[k]);
        }
      }
    }
    if (per_unit > 1) {
      s_ml[warp][lane][0] = m_run;
      s_ml[warp][lane][1] = l_run;
#pragma unroll
      for (int i = 0; i < kQuads; ++i) s_o[warp][i][lane] = o[i];
      __syncthreads();
      if (sub == 0) {
        for (int x = warp + 1; x < warp + per_unit; ++x) {
          float4 v[kQuads];
#pragma unroll
          for (int i = 0; i < kQuads; ++i) v[i] = s_o[x][i][lane];
          fold(s_ml[x][lane][0], s_ml[x][lane][1], v);
        }
      }
    }
    if (sub == 0 && row < rows) {
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      const int token = row / p.G;
      T* dst = static_cast<T*>(p.out) +
               (static_cast<size_t>(p.cu_q[s] + tok0 + token) * p.n_q + kvh * p.G + row - token * p.G) * D +
               cu * kMergeCols;
      uint32_t packed[2 * kQuads];
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        packed[2 * i] = Elt<T>::pack(o[i].x * inv, o[i].y * inv);
        packed[2 * i + 1] = Elt<T>::pack(o[i].z * inv, o[i].w * inv);
      }
      uint4* d4 = reinterpret_cast<uint4*>(dst);
#pragma unroll
      for (int i = 0; i < kQuads / 2; ++i) {
        d4[i] = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
      }
    }
    if (per_unit > 1) __syncthreads();
  }
}

// ── host side ────────────────────────────────────────────────────────────────

bool tree_shape_ok(int n_q, int n_kv, int D) {
  return (D == 64 || D == 128) && n_kv > 0 && n_kv <= 64 && n_q > 0 && n_q % n_kv == 0 &&
         n_q / n_kv <= 16;
}

struct TreeLayout {
  int part_rows;
  size_t records, ml, o, total;
};

// Contexts of at most kWholeTiles key tiles are not cut into pieces.
bool tree_whole(int max_blocks) { return max_blocks <= kWholeTiles * kTtPages; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

TreeLayout tree_layout(int max_q_len, int n_q, int n_kv, int D, int n_cta) {
  const int G = n_q / n_kv;
  const int tpt = kTtRows / G;
  const int tokens = max_q_len < tpt ? (max_q_len > 0 ? max_q_len : 1) : tpt;
  TreeLayout l;
  l.part_rows = (tokens * G + 31) / 32 * 32;
  l.records = 0;
  l.ml = align256(static_cast<size_t>(n_cta) * 8 * sizeof(int));
  l.o = l.ml + align256(static_cast<size_t>(n_cta) * 2 * l.part_rows * sizeof(float2));
  l.total = l.o + align256(static_cast<size_t>(n_cta) * 2 * l.part_rows * D * sizeof(float));
  return l;
}

template <typename... KArgs, typename... Args>
cudaError_t tree_launch(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t s,
                        Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename T, int D>
int launch_tree(const CUtensorMap& kv_map, const CUtensorMap& q_map, const TreeParams& p, int sms,
                cudaStream_t s) {
  using Shape = TreeShape<D>;
  static std::once_flag flags[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(VMPS_ERR_CUDA, "device index %d", dev);
  std::call_once(flags[dev], [] {
    cudaFuncSetAttribute(paged_tree_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         Shape::kFixedBytes + (kTtMaxSeqs + 1) * static_cast<int>(sizeof(int)));
  });
  const size_t smem = Shape::kFixedBytes + static_cast<size_t>(p.num_seqs + 1) * sizeof(int);
  cudaError_t e = tree_launch(paged_tree_kernel<T, D>, p.n_cta, kTtThreads, smem, s, kv_map, q_map, p);
  if (e == cudaSuccess && !p.whole) {
    e = tree_launch(paged_tree_merge_kernel<T, D>, kMergeBlocksPerSm * sms, kMergeThreads, 0, s, p);
  }
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "paged_tree_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" size_t vmps_paged_tree_attention_workspace_bytes(int num_seqs, int max_q_len, int n_q,
                                                            int n_kv, int head_dim,
                                                            int max_blocks_per_seq, int dtype) {
  if (num_seqs <= 0 || max_q_len <= 0 || max_q_len > kTtMaxQLen ||
      (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) ||
      !tree_shape_ok(n_q, n_kv, head_dim) || tree_whole(max_blocks_per_seq)) {
    return 0;
  }
  int sms = 0;
  if (device_sm_count(&sms)) return 0;
  return tree_layout(max_q_len, n_q, n_kv, head_dim, sms * kTtCtasPerSm).total;
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
  if (!tree_shape_ok(n_q, n_kv, head_dim)) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: n_q=%d n_kv=%d head_dim=%d not supported (head_dim 64/128, n_kv <= 64, "
                "n_q/n_kv a whole number up to 16)",
                what, n_q, n_kv, head_dim);
  }
  // The plan sums a row tile's tiles over all sequences in 31 bits.
  const long long max_tiles = (static_cast<long long>(max_blocks_per_seq) + kTtPages - 1) / kTtPages;
  if (num_seqs > kTtMaxSeqs || max_q_len > kTtMaxQLen || max_blocks_per_seq > (1 << 24) ||
      num_blocks > (1 << 29) ||
      num_seqs * (max_tiles * kTileWeight + kSegWeight) > 0x7fffffffLL) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: num_seqs=%d max_q_len=%d max_blocks=%d (num_seqs <= %d, max_q_len <= %d, "
                "max_blocks <= 2^24, num_seqs * max_blocks < 2^31, num_blocks <= 2^29)",
                what, num_seqs, max_q_len, max_blocks_per_seq, kTtMaxSeqs, kTtMaxQLen);
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
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  TreeParams p;
  p.n_cta = sms * kTtCtasPerSm;
  if (p.n_cta > kMaxCtas) return fail(VMPS_ERR_UNSUPPORTED, "%s: %d SMs", what, sms);
  const TreeLayout wl = tree_layout(max_q_len, n_q, n_kv, head_dim, p.n_cta);
  const bool whole = tree_whole(max_blocks_per_seq);
  // One that is given has to do for any context, one that is not needed may be missing.
  if (workspace ? workspace_bytes < wl.total : !whole) {
    return fail(VMPS_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, workspace_bytes,
                wl.total);
  }
  if (reinterpret_cast<uintptr_t>(workspace) & 255) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", what);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;

  const CUtensorMapDataType tdt =
      dtype == VMPS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t e = 2;
  const int G = n_q / n_kv;
  // Pool as {d, token, kv head, (block, K|V)}: a box [64][16][1][1] is one
  // page of one head, 16 rows of 128 bytes.
  CUtensorMap kv_map;
  {
    const uint64_t dims[4] = {(uint64_t)head_dim, kPage, (uint64_t)n_kv, (uint64_t)2 * num_blocks};
    const uint64_t strides[3] = {(uint64_t)n_kv * head_dim * e, (uint64_t)head_dim * e,
                                 (uint64_t)kPage * n_kv * head_dim * e};
    const uint32_t box[4] = {64, kPage, 1, 1};
    if (int rc = encode_tiled(&kv_map, tdt, 4, const_cast<void*>(pool), dims, strides, box,
                              CU_TENSOR_MAP_SWIZZLE_128B)) {
      return rc;
    }
  }
  // Queries as {d, head, row}: a box [64][G][tokens] is the rows (token-major,
  // head-minor) of one 64-column chunk of a row tile.
  p.tokens_per_tile = kTtRows / G;
  p.box_tokens = max_q_len < p.tokens_per_tile ? max_q_len : p.tokens_per_tile;
  CUtensorMap q_map;
  {
    const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)n_q, (uint64_t)total_q};
    const uint64_t strides[2] = {(uint64_t)head_dim * e, (uint64_t)q_row_stride * e};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)p.box_tokens};
    if (int rc = encode_tiled(&q_map, tdt, 3, const_cast<void*>(q), dims, strides, box,
                              CU_TENSOR_MAP_SWIZZLE_128B)) {
      return rc;
    }
  }
  p.out = out;
  p.pool = pool;
  p.block_tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.seq_lens = seq_lens;
  p.q_lens = q_lens;
  p.cu_q = cu_q;
  p.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  p.mask_words = mask_words;
  p.max_blocks = max_blocks_per_seq;
  p.num_seqs = num_seqs;
  p.total_q = total_q;
  p.max_q_len = max_q_len;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.G = G;
  p.num_blocks = num_blocks;
  p.row_tiles = (max_q_len + p.tokens_per_tile - 1) / p.tokens_per_tile;
  p.whole = whole ? 1 : 0;
  p.part_rows = wl.part_rows;
  p.scale_log2 = scale * 1.4426950408889634f;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.records = reinterpret_cast<int*>(ws + wl.records);
  p.part_ml = reinterpret_cast<float2*>(ws + wl.ml);
  p.part_o = reinterpret_cast<float4*>(ws + wl.o);
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VMPS_DTYPE_F16) {
    return head_dim == 64 ? launch_tree<__half, 64>(kv_map, q_map, p, sms, s)
                          : launch_tree<__half, 128>(kv_map, q_map, p, sms, s);
  }
  return head_dim == 64 ? launch_tree<__nv_bfloat16, 64>(kv_map, q_map, p, sms, s)
                        : launch_tree<__nv_bfloat16, 128>(kv_map, q_map, p, sms, s);
}
