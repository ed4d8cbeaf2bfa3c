// Kernel 11: decode attention over the 8-bit paged cache, one query token per
// sequence.
//
//   out[i][h] = softmax_t(scale * q[i][h] . K[t]) . V[t],  K, V = code * scale
//
// What bounds it: the codes' bytes from HBM (4 G operations per K and V code
// byte pair, G query heads a kv head).
//
//  * Work: tiles of 2 TG pages of HPC kv heads for HPC * TG = 8 consumer warps (HPC
//    2 where n_kv is even, else 1).  The tiles of all sequences are cut into equal
//    contiguous shares, one per CTA of a persistent grid, one CTA per SM
//    (cache8_plan.h), so that ragged batches and single long sequences both keep
//    every SM streaming.  Few heads a CTA mean few pieces: the first
//    kernel took 61.5 us for 32 ragged sequences with all 8 kv heads of a page in a
//    CTA and 40.4 with two.
//  * Four producer warps stream pages: a tiled TMA for the codes (K and V of HPC
//    heads, swizzled) and a bulk copy for their scales, into a ring of stages,
//    and the query rows of the next sequences into a ring of their own.
//  * A consumer warp takes two pages of one kv head a stage.  The G query heads
//    are the N side of m16n8k16 in fp16 with fp32 sums:
//        S^T[16 tok x 8 heads] = K . Q^T,   O^T[D x 8] += V^T . P^T
//    Codes become fp16 in registers, exactly: a byte under 0x64 is 1024 + byte
//    (int8: one xor per four codes, a byte permutation and a subtraction per
//    two), e4m3 has its conversion instruction.  ldmatrix hands a lane four
//    neighbouring bytes of a K row, which are taken as the MMA's k indices 2c,
//    2c+1, 2c+8, 2c+9 (Q is laid out to match), and with .trans two bytes of two
//    V rows, whose even and odd columns become rows g and g + 8 of the A operand:
//    the permutation that widens the codes also transposes them.
//  * K's scale multiplies the score.  V's multiplies the weight before its
//    rounding to fp16.  Weights are relative to a power of two 2^r per head and
//    warp that follows this product (its magnitude: a caller's scales may be
//    negative), so that the largest so far is 2^10 to 2^15 and what fp16 cannot
//    hold of small ones is 2^-35 of it, however large V is where the weights are
//    small.  Weights themselves, whose sums are fp32 and unrounded, are then
//    2^-111 (a product with V's largest possible scale) to 2^104; where V is so
//    small that its products want larger ones they stay at that, and rows of
//    V of 2^-100, the smallest that are stored, keep 17 bits.
//  * fp16 outputs get a second product with what that rounding left, without
//    which they were half as far again from the exact result as their own rounding
//    puts them (2.96e-4 in place of 2.08e-4 of the mean square).  It costs fp16 2.5 %
//    at 8 heads and 4.5 % at 16, in long runs, which the card's power holds back, 5 to
//    9 %.  bf16 outputs, whose own rounding is eight times the weights', would gain 1 %
//    of their error for as much, and do without.
//  * bf16 queries are scaled by a power of two per head, so that their largest
//    is in [2^13, 2^14), which fp16 holds as exactly as bf16 did but for values
//    below 2^-28 of it.
//  * At a sequence's end the warps of a kv head tell each other their references and sums,
//    write their outputs over the codes that they have just read and add up a part each.
//  * A cut sequence: every piece leaves its normalised output and the logarithm
//    of its weights' sum in fp32 and arrives on a counter; the last to arrive
//    joins, in two rounds where there are many pieces.  Sums are in a fixed order:
//    results do not depend on who is last.
#include <limits.h>

#include <mutex>
#include <type_traits>
#include <utility>

#include "cache8.cuh"
#include "cache8_plan.h"
#include "rows_overlap.h"
#include "vmps_abi_internal.h"

namespace vmps {
namespace {

constexpr int kMaxSeqs8 = 4096;
constexpr int kMaxKvHeads8 = 64;
constexpr int kMaxGroup8 = 16;
constexpr int kMaxStages8 = 8;
constexpr int kParts8 = 4;      // parts of a kv head's output, each joined by a warp of its own
constexpr int kWarps8 = 8;      // consumer warps of a CTA, at most
constexpr int kProducers8 = 4;  // producer warps: issuing a copy takes one about 100 clocks
constexpr int kMaxHeads8 = 8;   // kv heads of a CTA
// Pages that a warp takes of a tile.  Two share the waits and the checks of the scores and
// their products overlap: 4 x 131072 tokens 173.5 us for 176.0, 256 x 511..1537 96.8 for
// 102.8 (head size 128), 64 ragged sequences at head size 64 19.3 for 21.8.
constexpr int kPages8 = 2;
// The workspace's counters; the records start where the 16-bit decode kernel's
// do, so that one workspace serves both.
constexpr size_t kCounterBytes8 = size_t(128) << 10;
constexpr size_t kRecordsAt8 = size_t(1) << 20;
constexpr int kMostSmem8 = 220 << 10;  // dynamic shared memory of a CTA
constexpr float kLowest8 = -1e30f;  // the reference of weights where there were none
// Logarithm of the largest weight times V's scale after the reference has been raised (which
// it is when that has grown by 4), V's scales counted from 2^kLeastScale on: weights are at
// most 2^104 then, and the sum of 2^23 of them is finite.
constexpr float kMostProduct = 11.f, kLeastScale = -89.f;

struct Decode8Params {
  void* out;
  const void* q;
  int64_t q_stride;
  const float* scales;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  int max_blocks, num_seqs, n_kv, G, num_blocks;
  int hpc, tg;        // kv heads per CTA, pages per tile
  int stages;
  float scale_log2;   // scale * log2(e)
  int* group_counters;  // [n_cta][2][hpc][kParts8]
  int* top_counters;    // [n_cta][hpc][kParts8]
  // Records of the pieces (first half) and of the groups they are joined in.
  float* part_lse;      // [2][n_cta][2][hpc][NT][kParts8][4][2]
  float* part_o;        // [2][n_cta][2][hpc][NT * D / 16][32 lanes][4]
  int* err;
};

// A warp's note of a published piece of a cut sequence: its run of CTAs, the sequence and
// its kv head.
struct Piece8 {
  int c0, c1, s, kvh;
};

__device__ __forceinline__ int arrive_piece8(int* counter) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ uint32_t sub1152(uint32_t x) {
  uint32_t y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}

__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {
  uint32_t y;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n"
      : "=r"(y)
      : "r"(two));
  return y;
}

// Four code bytes -> two fp16 pairs: bytes 0, 1 and 2, 3 (kAlong) or bytes 0, 2
// and 1, 3.
template <bool kInt8, bool kAlong>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& first, uint32_t& second) {
  if constexpr (kInt8) {
    w ^= 0x80808080u;  // code + 128
    first = sub1152(__byte_perm(w, 0x64646464u, kAlong ? 0x4140 : 0x4240));
    second = sub1152(__byte_perm(w, 0x64646464u, kAlong ? 0x4342 : 0x4341));
  } else {
    if (!kAlong) w = __byte_perm(w, 0u, 0x3120);
    first = e4m3_pair(w);
    second = e4m3_pair(w >> 16);
  }
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What rounding a and b to fp16 (`two`) left of them.
__device__ __forceinline__ uint32_t remainder(float a, float b, uint32_t two) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
  return Elt<__half>::pack(a - f.x, b - f.y);
}

// Exponent of x >= 0 (the whole number in the low bits of 2^23).
__device__ __forceinline__ float exponent(float x) {
  return __uint_as_float((__float_as_uint(x) >> 23) | 0x4b000000u) - (8388608.f + 127.f);
}

// Joins part `part` (M m-tiles) of n-tile nt of `count` records (from `base` on, every
// `step`-th CTA's from `cta` on, slot 1 in CTA c0, 0 in the others): the normalised output
// in o, the logarithm of the weights' sum in lse.  The loads of a batch of records are in
// flight at once.
template <int D, int NT, int M>
__device__ __forceinline__ void join_records(const Decode8Params& p, size_t base, int cta, int step,
                                             int count, int c0, int h, int nt, int part, int lane,
                                             float (&lse)[2], float (&o)[M][4]) {
  constexpr int KS = D / 16;
  constexpr int kBatch = 8;
  const int c = lane & 3;
  // Lanes whose heads are padding (nothing was stored for them) read their neighbour's.
  const int from = nt * 8 + 2 * c < p.G ? lane : lane & ~3;
  const float2* ml = reinterpret_cast<const float2*>(p.part_lse) + (nt * kParts8 + part) * 4 + c;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) + (nt * KS + part * M) * 32 + from;
  float top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.f, sum1 = 0.f;
#pragma unroll
  for (int i = 0; i < M; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  for (int k0 = 0; k0 < count; k0 += kBatch) {
    float2 z[kBatch];
    float4 x[kBatch][M];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int b = cta + min(k0 + k, count - 1) * step;
      const size_t rec = base + (static_cast<size_t>(b) * 2 + (b == c0 ? 1 : 0)) * p.hpc + h;
      z[k] = __ldcg(ml + rec * NT * kParts8 * 4);
#pragma unroll
      for (int i = 0; i < M; ++i) x[k][i] = __ldcg(po + (rec * NT * KS + i) * 32);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (k0 + k >= count) z[k] = make_float2(-INFINITY, -INFINITY);
    }
    float t0 = top0, t1 = top1;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      t0 = fmaxf(t0, z[k].x);
      t1 = fmaxf(t1, z[k].y);
    }
    // -inf alone: nothing so far, and no factor that would be NaN.
    const float a0 = t0 == top0 ? 1.f : fast_exp2(top0 - t0);
    const float a1 = t1 == top1 ? 1.f : fast_exp2(top1 - t1);
    top0 = t0;
    top1 = t1;
    sum0 *= a0;
    sum1 *= a1;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      o[i][0] *= a0;
      o[i][1] *= a1;
      o[i][2] *= a0;
      o[i][3] *= a1;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w0 = z[k].x == -INFINITY ? 0.f : fast_exp2(z[k].x - top0);
      const float w1 = z[k].y == -INFINITY ? 0.f : fast_exp2(z[k].y - top1);
      sum0 += w0;
      sum1 += w1;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        o[i][0] = fmaf(w0, x[k][i].x, o[i][0]);
        o[i][1] = fmaf(w1, x[k][i].y, o[i][1]);
        o[i][2] = fmaf(w0, x[k][i].z, o[i][2]);
        o[i][3] = fmaf(w1, x[k][i].w, o[i][3]);
      }
    }
  }
  const float r0 = __fdividef(1.f, sum0), r1 = __fdividef(1.f, sum1);
  lse[0] = top0 + __log2f(sum0);
  lse[1] = top1 + __log2f(sum1);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    o[i][0] *= r0;
    o[i][1] *= r1;
    o[i][2] *= r0;
    o[i][3] *= r1;
  }
}

// M m-tiles (from mt on) of n-tile nt of the output rows of a kv head, from O^T fragments
// (rows g, g + 8 of an m-tile: elements 16 mt + 2g and the next; columns 2c, 2c + 1: heads).
template <typename T, int D, int M>
__device__ __forceinline__ void store_rows(T* rows, int G, int nt, int mt, int lane,
                                           const float (&o)[M][4]) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int n = nt * 8 + 2 * c + e;
    if (n >= G) continue;
    uint32_t* dst = reinterpret_cast<uint32_t*>(rows + n * D) + mt * 8 + g;
#pragma unroll
    for (int i = 0; i < M; ++i) dst[i * 8] = Elt<T>::pack(o[i][e], o[i][2 + e]);
  }
}

// The same into part `part` of a record, which has its own copy of the lse.
template <int D, int NT, int M>
__device__ __forceinline__ void store_record(const Decode8Params& p, size_t rec, int nt, int part,
                                             int lane, const float (&lse)[2], const float (&o)[M][4]) {
  if (nt * 8 + 2 * (lane & 3) < p.G) {
    float4* po =
        reinterpret_cast<float4*>(p.part_o) + ((rec * NT + nt) * (D / 16) + part * M) * 32 + lane;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      __stcg(po + i * 32, make_float4(o[i][0], o[i][1], o[i][2], o[i][3]));
    }
  }
  if (lane < 4) {
    __stcg(reinterpret_cast<float2*>(p.part_lse) + ((rec * NT + nt) * kParts8 + part) * 4 + lane,
           make_float2(lse[0], lse[1]));
  }
}

template <int D, int NT>
constexpr bool kRegroup8 = D == 128 && NT == 2;

template <typename T, int D, int NT, bool kInt8>
__global__ void __launch_bounds__(32 * (kProducers8 + kWarps8), 1)
decode8_kernel(const __grid_constant__ CUtensorMap tmap, const Decode8Params p) {
  constexpr int KS = D / 16;
  constexpr bool kF16 = std::is_same<T, __half>::value;
  __shared__ uint64_t full_bar[kMaxStages8];
  __shared__ uint64_t empty_bar[kMaxStages8];
  __shared__ uint64_t q_full[kMaxStages8 + 1];
  __shared__ uint64_t q_empty[kMaxStages8 + 1];
  // What a warp tells the others of its kv head at a segment's end: references and sums of heads
  // 2c, 2c + 1.  Two segments' worth: a warp can be writing the next one's
  // while another still reads.
  __shared__ float4 hand_ml_of[2][kWarps8][NT][4];
  __shared__ volatile int s_abort;
  __shared__ int warp_sum[kProducers8 + kWarps8];
  __shared__ C8Pos share[2];
  __shared__ Piece8 pieces_of[kWarps8][2];
  extern __shared__ uint8_t dyn_smem[];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.num_seqs, hpc = p.hpc, TG = p.tg, stages = p.stages;
  const int page_bytes = 2 * hpc * kCachePage * D;
  constexpr int PP = kPages8;
  const int TP = TG * PP;  // pages of a tile
  const int stage_bytes = TP * page_bytes;
  const int scale_bytes = hpc * 2 * kCachePage * 4;  // of one page
  constexpr int kQRow = D * 2 + 16;                  // a query row, padded: other banks
  const int q_bytes = hpc * p.G * kQRow;
  const int q_slots = stages + 1;

  // [ring][scales][query rows][prefix sums][lengths]
  const uint32_t base = smem_u32(dyn_smem);
  uint8_t* ring = dyn_smem + (((base + 1023u) & ~1023u) - base);
  float* ring_scales = reinterpret_cast<float*>(ring + stages * stage_bytes);
  uint8_t* q_ring = reinterpret_cast<uint8_t*>(ring_scales + stages * TP * scale_bytes / 4);
  int* wpref = reinterpret_cast<int*>(q_ring + q_slots * q_bytes);
  int* lens = wpref + n + 1;

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full_bar[i], kProducers8);
      mbar_init(&empty_bar[i], hpc * TG);
    }
    for (int i = 0; i < q_slots; ++i) {
      mbar_init(&q_full[i], kProducers8);
      mbar_init(&q_empty[i], hpc * TG);
    }
    fence_mbar_init();
  }
  chain_link();

  // ── the plan: lengths, prefix sums of their weights, this CTA's share ───────
  // Every thread owns `per` sequences; those in which the share begins and ends
  // are found by their owners.
  const int tile_shift = 31 - __clz(TP * kCachePage), tile_tokens = 1 << tile_shift;
  C8Shape sh;
  sh.num_seqs = n;
  sh.groups = p.n_kv / hpc;
  sh.n_cta = gridDim.x;
  {
    const int per = n <= blockDim.x ? 1 : (n + blockDim.x - 1) / blockDim.x;
    const int lo = min(n, tid * per), hi = min(n, lo + per);
    int sum = 0;
    for (int s = lo; s < hi; ++s) {
      int len = p.seq_lens[s];
      if (len <= 0) len = 0;
      if ((len + kCachePage - 1LL) / kCachePage > p.max_blocks) {
        if (blockIdx.x == 0) set_error(p.err, kDevErrSeqLen);
        len = p.max_blocks * kCachePage;
      }
      lens[s] = len;
      sum += c8_weight(c8_tiles(len, tile_shift));
    }
    int incl = sum;
#pragma unroll
    for (int sft = 1; sft < 32; sft <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, sft);
      if (lane >= sft) incl += y;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int run = incl - sum, total = 0;
    for (int x = 0; x < static_cast<int>(blockDim.x >> 5); ++x) {
      const int y = warp_sum[x];
      if (x < warp) run += y;
      total += y;
    }
    sh.chunk = c8_chunk(total, sh.groups, sh.n_cta);
    const long long w0 = static_cast<long long>(blockIdx.x) * sh.chunk;
    C8Cut cut[2] = {c8_cut(total, sh.groups, w0), c8_cut(total, sh.groups, w0 + sh.chunk)};
    if (tid == 0) {
      wpref[0] = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (cut[e].hg == sh.groups) share[e] = C8Pos{sh.groups, 0, 0};
      }
    }
    for (int s = lo; s < hi; ++s) {
      const int before = run;
      run += c8_weight(c8_tiles(lens[s], tile_shift));
      wpref[s + 1] = run;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (cut[e].hg < sh.groups && before <= cut[e].at && cut[e].at < run) {
          share[e] = C8Pos{cut[e].hg, s, c8_tile_at(cut[e].at - before)};
        }
      }
    }
    __syncthreads();
  }
  const C8Pos begin = share[0], end = share[1];
  C8Walk w;
  w.start(wpref, sh, begin, end);

  // At head size 128 the sums of 16 query heads take more registers than 12 warps have each:
  // the producers' warpgroup hands some to the two of the consumers (128 * 56 + 256 * 224 =
  // 384 * 168, what the block was launched with).
  if constexpr (kRegroup8<D, NT>) {
    if (warp < kProducers8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    }
  }
  if (warp < kProducers8) {
    // ── producers ────────────────────────────────────────────────────────────
    // Block-table entries are fetched 32 pages ahead of their use.
    if (lane == 0) prefetch_tmap(&tmap);
    int pg = 0, pg_end = 0;
    bool fresh = false;  // the next batch is a segment's first
    auto enter = [&]() {
      pg = w.j0 * TP;
      pg_end = min(w.j1 * TP, (lens[w.s] - 1) / kCachePage + 1);
      fresh = true;
    };
    auto fetch = [&](int& hg, int& count, int& phys, int& first_of) {
      count = 0;
      if (!w.valid) return;
      hg = w.hg;
      first_of = fresh ? w.s : -1;
      fresh = false;
      count = min(32, pg_end - pg);
      phys = 0;
      if (lane < count) phys = p.block_tables[static_cast<int64_t>(w.s) * p.max_blocks + pg + lane];
      pg += count;
      if (pg == pg_end) {
        w.next(wpref, sh, end);
        if (w.valid) enter();
      }
    };
    if (w.valid) enter();
    int hg = 0, count, phys = 0, seq = -1, hg2 = 0, count2, phys2 = 0, seq2 = -1;
    fetch(hg, count, phys, seq);
    int stage = 0, q_slot = 0;
    uint32_t parity = 1, q_parity = 1;
    while (count > 0) {
      fetch(hg2, count2, phys2, seq2);
      const bool bad = phys < 0 || phys >= p.num_blocks;
      if (bad) set_error(p.err, kDevErrBlockRange);
      // Such a page's codes read as zeros (the tensor map's bounds), its scales as block 0's.
      const float* src = p.scales + (static_cast<size_t>(bad ? 0 : phys) * p.n_kv + hg * hpc) * 2 * kCachePage;
      if (bad) phys = p.num_blocks;
      for (int k = 0; k < count; k += TP) {
        const int np = min(TP, count - k);
        const bool ok = !s_abort && mbar_wait(&empty_bar[stage], parity, p.err);
        if (!__all_sync(0xffffffffu, ok)) {
          s_abort = 1;
          return;
        }
        // This warp's pages of the tile: every kProducers8-th.
        const int mine = (np - warp + kProducers8 - 1) / kProducers8;
        if (lane == 0) {
          if (mine > 0) {
            mbar_arrive_expect_tx(&full_bar[stage], mine * (page_bytes + scale_bytes));
          } else {
            mbar_arrive(&full_bar[stage]);
          }
        }
        __syncwarp();
        const int i = lane - k;
        if (i >= 0 && i < np && i % kProducers8 == warp) {
          tma_load_4d(ring + stage * stage_bytes + i * page_bytes, &tmap, &full_bar[stage], 0, 0,
                      D == 64 && hpc % 2 == 0 ? hg * (hpc / 2) : hg * hpc, 2 * phys);
          bulk_load(ring_scales + (stage * TP + i) * (scale_bytes / 4), src, scale_bytes,
                    &full_bar[stage]);
        }
        if (++stage == stages) {
          stage = 0;
          parity ^= 1;
        }
        if (k == 0 && seq >= 0) {
          // The segment's query rows, every kProducers8-th by this warp, behind its first pages.
          const bool ok = !s_abort && mbar_wait(&q_empty[q_slot], q_parity, p.err);
          if (!__all_sync(0xffffffffu, ok)) {
            s_abort = 1;
            return;
          }
          const int rows = hpc * p.G, mine = (rows - warp + kProducers8 - 1) / kProducers8;
          if (lane == 0) {
            if (mine > 0) {
              mbar_arrive_expect_tx(&q_full[q_slot], mine * D * 2);
            } else {
              mbar_arrive(&q_full[q_slot]);
            }
          }
          __syncwarp();
          if (lane < mine) {
            const int row = warp + lane * kProducers8;
            bulk_load(q_ring + q_slot * q_bytes + row * kQRow,
                      static_cast<const T*>(p.q) + seq * p.q_stride +
                          (static_cast<int64_t>(hg) * hpc * p.G + row) * D,
                      D * 2, &q_full[q_slot]);
          }
          if (++q_slot == q_slots) {
            q_slot = 0;
            q_parity ^= 1;
          }
        }
      }
      hg = hg2;
      count = count2;
      phys = phys2;
      seq = seq2;
    }
    return;
  }

  // ── consumers ─────────────────────────────────────────────────────────────
  const int cw = warp - kProducers8;
  const int h = cw % hpc, tg = cw / hpc;
  const int g = lane >> 2, c = lane & 3;
  T* out = static_cast<T*>(p.out);
  const int n_q = p.n_kv * p.G;
  for (int s = blockIdx.x; s < n; s += gridDim.x) {  // rows of empty sequences
    if (lens[s] > 0) continue;
    uint4* o4 = reinterpret_cast<uint4*>(out + static_cast<int64_t>(s) * n_q * D);
    for (int e = tid - 32 * kProducers8; e < n_q * D / 8; e += blockDim.x - 32 * kProducers8) o4[e] = make_uint4(0u, 0u, 0u, 0u);
  }

  if (cw >= hpc * TG) return;  // (whole warpgroups are launched where registers change hands)

  // Where the tensor map's box and swizzle put 16-byte chunk `chunk` of this head's row of
  // token `tok` in a page (K; V is v_add further): rows of 128 bytes, at head size 64 of two
  // heads, or of 64 where n_kv is odd.
  const bool two = D == 64 && hpc % 2 == 0;
  auto place = [&](int tok, int chunk) -> uint32_t {
    if (D == 128) return h * (kCachePage * D) + tok * 128 + ((chunk ^ (tok & 7)) << 4);
    if (two) {
      return (h >> 1) * (kCachePage * 128) + tok * 128 + ((((h & 1) * 4 + chunk) ^ (tok & 7)) << 4);
    }
    return h * (kCachePage * D) + tok * 64 + ((chunk ^ ((tok >> 1) & 3)) << 4);
  };
  // This lane's ldmatrix row: token r (+ 8 for matrices 1 and 3), chunk 2 kk (+ 1 for matrices
  // 2 and 3).
  uint32_t off[D / 32];
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) {
    off[kk] = place((lane & 7) + ((lane >> 3) & 1) * 8, 2 * kk + (lane >> 4));
  }
  const uint32_t k_base = smem_u32(ring) + tg * page_bytes;
  const uint32_t v_add = hpc * kCachePage * D;
  const float* my_scales = ring_scales + (tg * hpc + h) * 2 * kCachePage + g;

  Piece8* pend = pieces_of[cw];
  int n_pend = 0;
  // The counter a piece arrives on, and how many do.
  auto counter_of = [&](int i, int& members) -> int* {
    const int pieces = pend[i].c1 - pend[i].c0 + 1;
    const int size = c8_join_group(pieces);
    const int first = (static_cast<int>(blockIdx.x) - pend[i].c0) / size * size;
    members = min(size, pieces - first);
    const int lead = pend[i].c0 + first;
    return p.group_counters +
           ((static_cast<size_t>(lead) * 2 + (first == 0 ? 1 : 0)) * hpc + h) * kParts8 + tg;
  };

  // The warps of a kv head, at one point.
  auto together = [&]() { named_barrier_sync(1 + h, TG * 32); };
  constexpr int M = KS / kParts8;  // m-tiles that a warp takes of a kv head's output at a time

  int stage = 0, q_slot = 0, turn = 0;
  uint32_t parity = 0, q_parity = 0;
  for (C8Walk following; w.valid; w = following, turn ^= 1) {
    following = w;  // worked out here, where the first tile is waited for anyway
    following.next(wpref, sh, end);
    const int s = w.s, kvh = w.hg * hpc + h, len = lens[s];
    if (!s_abort && !mbar_wait(&q_full[q_slot], q_parity, p.err)) s_abort = 1;
    // Q^T as the B operand: k indices 2c, 2c+1 and 2c+8, 2c+9 of step ks are elements
    // 16 ks + 4c .. + 3 of head g.
    uint32_t qf[NT][KS][2];
    float fac[NT][2];  // of heads 2c, 2c + 1: score -> log2 units
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + g;
      const uint8_t* row =
          q_ring + q_slot * q_bytes + (h * p.G + (head < p.G ? head : 0)) * kQRow + 8 * c;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 32 * ks);
        qf[nt][ks][0] = head < p.G ? v.x : 0u;
        qf[nt][ks][1] = head < p.G ? v.y : 0u;
      }
      float mine = p.scale_log2;
      if constexpr (!kF16) {
        uint32_t two = 0;  // the largest magnitudes of even and odd elements
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int e = 0; e < 2; ++e) two = __vmaxu2(two, qf[nt][ks][e] & 0x7fff7fffu);
        }
        uint32_t top = max(two << 16, two & 0xffff0000u);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = 13 - (static_cast<int>(top >> 23) - 127);
        if (top >= 0x7f800000u || top == 0) e = 0;
        e = max(-100, min(100, e));
        const float up = pow2(e);
        mine *= pow2(-e);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = qf[nt][ks][i];
            qf[nt][ks][i] = Elt<__half>::pack(__uint_as_float(x << 16) * up,
                                              __uint_as_float(x & 0xffff0000u) * up);
          }
        }
      }
      fac[nt][0] = __shfl_sync(0xffffffffu, mine, 8 * c);
      fac[nt][1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
    }

    __syncwarp();
    if (lane == 0) mbar_arrive(&q_empty[q_slot]);
    if (++q_slot == q_slots) {
      q_slot = 0;
      q_parity ^= 1;
    }

    float r[NT][2], l[NT][2], o[NT][KS][4];  // r: the weights' reference, a whole number
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      r[nt][0] = r[nt][1] = kLowest8;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }

    // One page or PP of a tile: `live` tokens from the first on, the others TG pages further
    // each (all but the last whole).
    auto work = [&](auto pages_tag, int live) {
      constexpr int P = decltype(pages_tag)::value;
      const uint32_t kb = k_base + stage * stage_bytes;
      const float* sc = my_scales + stage * TP * (scale_bytes / 4);
      const int last_live = live - (P - 1) * TG * kCachePage;  // of the last page
      const bool tail = last_live < kCachePage;
      float x[P][NT][4], ks0[P], ks1[P], vs0[P], vs1[P], lv0[P], lv1[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float* si = sc + i * TG * (scale_bytes / 4);
        ks0[i] = si[0];
        ks1[i] = si[8];
        vs0[i] = si[16];
        vs1[i] = si[24];
        lv0[i] = fmaxf(fast_log2(fabsf(vs0[i])), kLeastScale);
        lv1[i] = fmaxf(fast_log2(fabsf(vs1[i])), kLeastScale);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) x[i][nt][0] = x[i][nt][1] = x[i][nt][2] = x[i][nt][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          uint32_t a[4], b[4], d[4];
          ldmatrix_x4(a, kb + i * TG * page_bytes + off[kk]);
          widen<kInt8, true>(a[0], b[0], b[2]);
          widen<kInt8, true>(a[1], b[1], b[3]);
          widen<kInt8, true>(a[2], d[0], d[2]);
          widen<kInt8, true>(a[3], d[1], d[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Mma<__half>::run(x[i][nt], b, qf[nt][2 * kk][0], qf[nt][2 * kk][1]);
            Mma<__half>::run(x[i][nt], d, qf[nt][2 * kk + 1][0], qf[nt][2 * kk + 1][1]);
          }
        }
      }
      // Scores in log2 units less r; behind the length, whatever the slots hold, none.
      float y[P][NT][4];
      auto score = [&]() {
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            y[i][nt][0] = fmaf(x[i][nt][0], fac[nt][0] * ks0[i], -r[nt][0]);
            y[i][nt][1] = fmaf(x[i][nt][1], fac[nt][1] * ks0[i], -r[nt][1]);
            y[i][nt][2] = fmaf(x[i][nt][2], fac[nt][0] * ks1[i], -r[nt][0]);
            y[i][nt][3] = fmaf(x[i][nt][3], fac[nt][1] * ks1[i], -r[nt][1]);
          }
        }
        if (tail) {
          if (g >= last_live) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) y[P - 1][nt][0] = y[P - 1][nt][1] = -INFINITY;
            vs0[P - 1] = 0.f;
          }
          if (g + 8 >= last_live) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) y[P - 1][nt][2] = y[P - 1][nt][3] = -INFINITY;
            vs1[P - 1] = 0.f;
          }
        }
      };
      score();
      float most = -INFINITY;  // logarithm of the largest product
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float y0 = fmaxf(y[i][0][0], y[i][0][1]), y1 = fmaxf(y[i][0][2], y[i][0][3]);
#pragma unroll
        for (int nt = 1; nt < NT; ++nt) {
          y0 = fmaxf(y0, fmaxf(y[i][nt][0], y[i][nt][1]));
          y1 = fmaxf(y1, fmaxf(y[i][nt][2], y[i][nt][3]));
        }
        most = fmaxf(most, fmaxf(y0 + lv0[i], y1 + lv1[i]));
      }
      if (__any_sync(0xffffffffu, most > kMostProduct + 4.f)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float to = -INFINITY;
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float s0 = x[i][nt][e] * (fac[nt][e] * ks0[i]);
              const float s1 = x[i][nt][2 + e] * (fac[nt][e] * ks1[i]);
              // (Scales are finite up to 2^128; infinite ones make infinite products.)
              if (i < P - 1 || g < last_live) to = fmaxf(to, s0 + fminf(lv0[i], 128.f));
              if (i < P - 1 || g + 8 < last_live) to = fmaxf(to, s1 + fminf(lv1[i], 128.f));
            }
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, b));
            to = fmaxf(r[nt][e], ceilf(to - kMostProduct));
            const float down = fast_exp2(r[nt][e] - to);
            r[nt][e] = to;
            l[nt][e] *= down;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
              o[nt][mt][e] *= down;
              o[nt][mt][2 + e] *= down;
            }
          }
        }
        score();
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        uint32_t pb[NT][2];  // rounded weights
        [[maybe_unused]] uint32_t pl[NT][2];  // for fp16, what that left
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float p0 = fast_exp2(y[i][nt][0]), p1 = fast_exp2(y[i][nt][1]);
          const float p2 = fast_exp2(y[i][nt][2]), p3 = fast_exp2(y[i][nt][3]);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          // C fragment (row = token, col = head) -> B fragment (k = token, n = head).
          const float w0 = p0 * vs0[i], w1 = p1 * vs0[i], w2 = p2 * vs1[i], w3 = p3 * vs1[i];
          const uint32_t lo = Elt<__half>::pack(w0, w1), hi = Elt<__half>::pack(w2, w3);
          pb[nt][0] = movmatrix_trans(lo);
          pb[nt][1] = movmatrix_trans(hi);
          if constexpr (kF16) {
            pl[nt][0] = movmatrix_trans(remainder(w0, w1, lo));
            pl[nt][1] = movmatrix_trans(remainder(w2, w3, hi));
          }
        }
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          uint32_t a[4], b[4], d[4];
          ldmatrix_x4_trans(a, kb + i * TG * page_bytes + v_add + off[kk]);
          if (!kInt8 && i == P - 1 && tail) {
            // e4m3 has NaN codes, and 0 * NaN is one: tokens 2c, 2c+1 and 2c+8, 2c+9.
            const uint32_t lo = (2 * c < last_live ? 0xffffu : 0u) |
                                (2 * c + 1 < last_live ? 0xffff0000u : 0u);
            const uint32_t hi = (2 * c + 8 < last_live ? 0xffffu : 0u) |
                                (2 * c + 9 < last_live ? 0xffff0000u : 0u);
            a[0] &= lo;
            a[1] &= hi;
            a[2] &= lo;
            a[3] &= hi;
          }
          widen<kInt8, false>(a[0], b[0], b[1]);
          widen<kInt8, false>(a[1], b[2], b[3]);
          widen<kInt8, false>(a[2], d[0], d[1]);
          widen<kInt8, false>(a[3], d[2], d[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Mma<__half>::run(o[nt][2 * kk], b, pb[nt][0], pb[nt][1]);
            Mma<__half>::run(o[nt][2 * kk + 1], d, pb[nt][0], pb[nt][1]);
            if constexpr (kF16) {
              Mma<__half>::run(o[nt][2 * kk], b, pl[nt][0], pl[nt][1]);
              Mma<__half>::run(o[nt][2 * kk + 1], d, pl[nt][0], pl[nt][1]);
            }
          }
        }
      }
    };

    int live = len - (w.j0 * TP + tg) * kCachePage;  // tokens from this warp's first page on
    for (int j = w.j0; j < w.j1; ++j, live -= tile_tokens) {
      // After a wait that gave up, the rest runs through without waiting: the barriers
      // between warps still meet.
      if (!mbar_try_wait(&full_bar[stage], parity) && !s_abort &&
          !mbar_wait(&full_bar[stage], parity, p.err)) {
        s_abort = 1;
      }
      if (PP > 1 && live > (PP - 1) * TG * kCachePage) {
        work(std::integral_constant<int, PP>{}, live);
      } else if (live > 0) {
        work(std::integral_constant<int, 1>{}, live);
      }
      if (j + 1 < w.j1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty_bar[stage]);
        if (++stage == stages) {
          stage = 0;
          parity ^= 1;
        }
      }
    }

    // ── the segment's end: the warps of a kv head put their sums together ─────
    const int active = min(TG, (len - 1) / kCachePage + 1 - w.j0 * TP);  // warps that had a page
    const bool whole = w.j0 == 0 && w.j1 == w.tiles;
    const bool alone = whole && active == 1;
    T* rows = out + (static_cast<int64_t>(s) * n_q + kvh * p.G) * D;
    // Bounds and sums first.
    float4(*hand_ml)[NT][4] = hand_ml_of[turn];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) {
        l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], b);
        l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], b);
      }
      if (g == 0) hand_ml[cw][nt][c] = make_float4(r[nt][0], r[nt][1], l[nt][0], l[nt][1]);
    }
    if (alone) {
      __syncwarp();
    } else {
      together();
    }
    float lse[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // Lane (g, c) looks at warp g's; the butterflies leave every lane with the same sums.
      float4 ml = make_float4(kLowest8, kLowest8, 0.f, 0.f);
      if (g < active) ml = hand_ml[g * hpc + h][nt][c];
      // A warp's sum may be far from 1: its exponent counts with the reference.  (What is lost
      // of the others' is below 2^-22 of the whole.)
      float top0 = ml.x + exponent(ml.z), top1 = ml.y + exponent(ml.w);
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) {
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, b));
        top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, b));
      }
      float sum0 = ml.z * fast_exp2(ml.x - top0), sum1 = ml.w * fast_exp2(ml.y - top1);
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) {
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, b);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, b);
      }
      lse[nt][0] = top0 + __log2f(sum0);
      lse[nt][1] = top1 + __log2f(sum1);
      // A cut piece whose weights are all zero (scores of -inf) adds nothing.
      const float r0 = !whole && sum0 == 0.f ? 0.f : __fdividef(1.f, sum0);
      const float r1 = !whole && sum1 == 0.f ? 0.f : __fdividef(1.f, sum1);
      const float a0 = fast_exp2(r[nt][0] - top0) * r0;
      const float a1 = fast_exp2(r[nt][1] - top1) * r1;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        o[nt][mt][0] *= a0;
        o[nt][mt][1] *= a1;
        o[nt][mt][2] *= a0;
        o[nt][mt][3] *= a1;
      }
    }
    if (alone) {
      if (tg == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) store_rows<T, D, KS>(rows, p.G, nt, 0, lane, o[nt]);
      }
    } else {
      // Then the output: each warp writes its share over the codes that it has just read (the
      // last tile's slot is given back after that), and adds up all warps' in M m-tiles.
      uint8_t* slot = ring + stage * stage_bytes;
      // A fragment of m-tile mt takes the head's chunks from 32 mt on, K's and then V's.
      auto chunk_of = [&](int mt) -> uint32_t {
        const int at = (mt % (KS / 2)) * 32 + lane;
        return (mt >= KS / 2 ? v_add : 0u) + place(at / (D / 16), at % (D / 16));
      };
      // Record of this CTA's end (slot 0) or start (slot 1) of a cut sequence.
      const size_t rec = (static_cast<size_t>(blockIdx.x) * 2 + (w.j0 == 0)) * hpc + h;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt > 0) together();  // the n-tile before has been read
        if (tg < active) {
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            *reinterpret_cast<float4*>(slot + tg * page_bytes + chunk_of(mt)) =
                make_float4(o[nt][mt][0], o[nt][mt][1], o[nt][mt][2], o[nt][mt][3]);
          }
          // The next tile's copy into this slot comes after these writes.  (Here, where no
          // global stores are under way that the fence would wait for.)
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        together();
        for (int mt = tg * M; mt < KS; mt += TG * M) {
          float x[M][4];
          float4 y[kWarps8][M];
#pragma unroll
          for (int i = 0; i < M; ++i) {
            const uint8_t* from = slot + chunk_of(mt + i);
#pragma unroll
            for (int t = 0; t < kWarps8; ++t) {
              y[t][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (t < active) y[t][i] = *reinterpret_cast<const float4*>(from + t * page_bytes);
            }
          }
#pragma unroll
          for (int i = 0; i < M; ++i) {
            x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
            for (int t = 0; t < kWarps8; ++t) {
              x[i][0] += y[t][i].x;
              x[i][1] += y[t][i].y;
              x[i][2] += y[t][i].z;
              x[i][3] += y[t][i].w;
            }
          }
          if (whole) {
            store_rows<T, D, M>(rows, p.G, nt, mt, lane, x);
          } else {
            store_record<D, NT, M>(p, rec, nt, mt / M, lane, lse[nt], x);
          }
        }
      }
    }
    // The slot goes back to the copies of the next tiles.
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty_bar[stage]);
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
    if (whole) continue;
    if (n_pend == 2) {  // the plan leaves a CTA two pieces at most
      set_error(p.err, kDevErrSeqLen);
      continue;
    }
    if (lane < 2) {
      (lane == 0 ? pend[n_pend].c0 : pend[n_pend].c1) =
          c8_owner(wpref, sh, w.hg, s, lane == 0 ? 0 : w.tiles - 1);
    }
    pend[n_pend].s = s;
    pend[n_pend].kvh = kvh;
    ++n_pend;
  }
  if (n_pend == 0 || tg >= kParts8) return;

  // ── joining cut sequences ─────────────────────────────────────────────────
  // The first kParts8 warps of a kv head join M m-tiles each, those that they stored of the
  // pieces: a warp waits for nobody.
  __syncwarp();  // every lane's stores before those lanes' releases
  int missing = -1;
  if (lane < n_pend) {
    int members;
    int* counter = counter_of(lane, members);
    missing = members - 1 - arrive_piece8(counter);
  }
  // Every lane's loads of other CTAs' records come after those lanes' acquires, and lane 0's
  // reset of a counter after the lane's arrival on it.
  __syncwarp();
  for (int i = 0; i < n_pend; ++i) {
    if (__shfl_sync(0xffffffffu, missing, i) != 0) continue;
    const int c0 = pend[i].c0, pieces = pend[i].c1 - c0 + 1;
    const int size = c8_join_group(pieces);
    const int first = (static_cast<int>(blockIdx.x) - c0) / size * size;
    T* rows = out + (static_cast<int64_t>(pend[i].s) * n_q + pend[i].kvh * p.G) * D;
    int members;
    int* counter = counter_of(i, members);
    if (lane == 0) *counter = 0;
    const size_t round2 = static_cast<size_t>(gridDim.x) * 2 * hpc;  // records after the pieces'
    float lse[2], x[M][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      join_records<D, NT, M>(p, 0, c0 + first, 1, members, c0, h, nt, tg, lane, lse, x);
      if (size == pieces) {
        store_rows<T, D, M>(rows, p.G, nt, tg * M, lane, x);
      } else {
        store_record<D, NT, M>(p, round2 + (static_cast<size_t>(c0 + first) * 2 + (first == 0)) * hpc + h,
                               nt, tg, lane, lse, x);
      }
    }
    if (size == pieces) continue;
    const int groups = (pieces + size - 1) / size;
    __syncwarp();
    int before = 0;
    if (lane == 0) {
      int* top = p.top_counters + (static_cast<size_t>(c0) * hpc + h) * kParts8 + tg;
      before = arrive_piece8(top);
      if (before == groups - 1) *top = 0;
    }
    __syncwarp();  // every lane's loads come after lane 0's acquire
    if (__shfl_sync(0xffffffffu, before, 0) != groups - 1) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      join_records<D, NT, M>(p, round2, c0, size, groups, c0, h, nt, tg, lane, lse, x);
      store_rows<T, D, M>(rows, p.G, nt, tg * M, lane, x);
    }
  }
}

// ── host side ────────────────────────────────────────────────────────────────

struct Decode8Config {
  int hpc, tg, nt, n_cta, stages;
  size_t smem, lse_at, o_at, workspace;
};

size_t align256_8(size_t x) { return (x + 255) & ~size_t(255); }

bool shape_ok8(int num_seqs, int n_q, int n_kv, int D) {
  return num_seqs >= 0 && num_seqs <= kMaxSeqs8 && n_kv > 0 && n_kv <= kMaxKvHeads8 && n_q > 0 &&
         n_q % n_kv == 0 && n_q / n_kv <= kMaxGroup8 && (D == 64 || D == 128);
}

// The launch for a shape (shape_ok8) on a device with `sms` SMs.
Decode8Config configure8(int num_seqs, int n_q, int n_kv, int D, int max_blocks, int sms) {
  Decode8Config cfg;
  // Two heads a CTA, so that a sequence is cut into few pieces and rows of a page are
  // read 2 D bytes at a time; more where no sequence has the pages for the other warps.
  cfg.nt = n_q / n_kv > 8 ? 2 : 1;
  cfg.tg = kWarps8 / 2;
  while (cfg.tg > 1 && cfg.tg / 2 * kPages8 >= max_blocks) cfg.tg /= 2;
  cfg.hpc = min(kMaxHeads8, kWarps8 / cfg.tg);
  while (cfg.hpc > 2 && cfg.hpc * (n_q / n_kv) > 32) --cfg.hpc;  // query rows in shared memory
  while (n_kv % cfg.hpc) --cfg.hpc;
  while (cfg.hpc * cfg.tg * 2 <= kWarps8 && cfg.tg * kPages8 < max_blocks) cfg.tg *= 2;
  cfg.n_cta = sms;
  const size_t stage =
      static_cast<size_t>(cfg.tg) * kPages8 * cfg.hpc * (2 * kCachePage * D + 2 * kCachePage * 4);
  const size_t q_slot = static_cast<size_t>(cfg.hpc) * (n_q / n_kv) * (2 * D + 16);
  const size_t rest = 1024 + q_slot + (2 * static_cast<size_t>(num_seqs) + 1) * 4;
  // Bytes in flight: three stages at head size 128 (4 x 131072 tokens 173.5 us, 176.8 with
  // two; 256 x 511..1537 96.8 and 104.3), four at 64 (16 x 1..8192 42.2 us, 44.5 with six and
  // 45.9 with two: what is in flight beyond the need makes the waits of the joins longer).
  const size_t most = D == 128 ? 208 << 10 : 160 << 10;
  cfg.stages = kMaxStages8;
  while (cfg.stages > 2 && (cfg.stages * stage > most ||
                            rest + cfg.stages * (stage + q_slot) > kMostSmem8)) {
    --cfg.stages;
  }
  cfg.smem = rest + cfg.stages * (stage + q_slot);
  const size_t recs = static_cast<size_t>(cfg.n_cta) * 2 * 2 * 2;
  cfg.lse_at = kRecordsAt8;
  cfg.o_at = cfg.lse_at + align256_8(recs * cfg.nt * kParts8 * 8 * sizeof(float));
  cfg.workspace = cfg.o_at + recs * cfg.nt * (D / 16) * 128 * sizeof(float);
  return cfg;
}

template <typename T, int D, int NT, bool kInt8>
int launch_decode8(const CUtensorMap& tmap, const Decode8Params& p, const Decode8Config& c,
                   cudaStream_t s) {
  static std::once_flag flags[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(VMPS_ERR_CUDA, "device index %d", dev);
  std::call_once(flags[dev], [] {
    cudaFuncSetAttribute(decode8_kernel<T, D, NT, kInt8>,
                         cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem8);
  });
  const cudaError_t e =
      launch_link(decode8_kernel<T, D, NT, kInt8>, true, dim3(c.n_cta),
                  dim3(32 * (kProducers8 + (kRegroup8<D, NT> ? kWarps8 : c.hpc * c.tg))), c.smem, s,
                  tmap, p);
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "paged_decode_attention_cache8: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
}

template <typename T, bool kInt8>
int dispatch_decode8(int D, const CUtensorMap& tmap, const Decode8Params& p, const Decode8Config& c,
                     cudaStream_t s) {
  if (D == 64) {
    return c.nt == 1 ? launch_decode8<T, 64, 1, kInt8>(tmap, p, c, s)
                     : launch_decode8<T, 64, 2, kInt8>(tmap, p, c, s);
  }
  return c.nt == 1 ? launch_decode8<T, 128, 1, kInt8>(tmap, p, c, s)
                   : launch_decode8<T, 128, 2, kInt8>(tmap, p, c, s);
}

}  // namespace
}  // namespace vmps

extern "C" size_t vmps_paged_decode_cache8_workspace_bytes(int num_seqs, int n_q, int n_kv,
                                                           int head_dim) {
  using namespace vmps;
  int sms = 0;
  if (!shape_ok8(num_seqs, n_q, n_kv, head_dim) || device_sm_count(&sms)) return 0;
  return configure8(num_seqs, n_q, n_kv, head_dim, INT_MAX, sms).workspace;
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
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (cache_format != VMPS_CACHE_INT8 && cache_format != VMPS_CACHE_E4M3) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: cache_format %d", what, cache_format);
  }
  if (block_size != kCachePage) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: block_size %d (only 16 is built)", what, block_size);
  }
  if (!shape_ok8(num_seqs, n_q, n_kv, head_dim)) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: num_seqs=%d n_q=%d n_kv=%d head_dim=%d not supported (num_seqs <= 4096, "
                "head_dim 64/128, n_kv <= 64, n_q/n_kv whole and at most 16)",
                what, num_seqs, n_q, n_kv, head_dim);
  }
  // Lengths, and the weights that the plan sums up, stay within 31 bits; a tensor
  // map's coordinates as well.
  if (max_blocks_per_seq > 0x7fffffff / kCachePage || num_blocks > 0x3fffffff ||
      static_cast<int64_t>(num_seqs) * c8_weight(max_blocks_per_seq) > 0x7fffffff) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: num_seqs=%d max_blocks=%d num_blocks=%d not supported",
                what, num_seqs, max_blocks_per_seq, num_blocks);
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
  const int64_t q_row = static_cast<int64_t>(n_q) * head_dim;
  if (rows_overlap(out, q_row * 2, q_row * 2, q, q_row_stride * 2, q_row * 2, num_seqs)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: out overlaps q", what);
  }
  if (!(scale > 0.f) || !(scale < 1e30f)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: scale %g", what, (double)scale);
  }
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const Decode8Config cfg = configure8(num_seqs, n_q, n_kv, head_dim, max_blocks_per_seq, sms);
  if (static_cast<size_t>(cfg.n_cta) * 3 * 2 * kParts8 * sizeof(int) > kCounterBytes8) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: %d SMs", what, sms);
  }
  if (!workspace || workspace_bytes < cfg.workspace) {
    return fail(VMPS_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, workspace_bytes,
                cfg.workspace);
  }
  if (reinterpret_cast<uintptr_t>(workspace) & 255) {
    return fail(VMPS_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", what);
  }
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  // The cache as {row, token, heads, (block, K|V)}, a row being 128 bytes of one head or,
  // at head size 64, of two (half as many lines for the copy engine; 64 bytes where n_kv is
  // odd): the box lands as [K|V][heads][token] rows, their 16-byte chunks swizzled.
  CUtensorMap tmap;
  const int per_row = head_dim == 64 && cfg.hpc % 2 == 0 ? 2 : 1;
  const uint64_t row = (uint64_t)per_row * head_dim;
  const uint64_t dims[4] = {row, (uint64_t)kCachePage, (uint64_t)n_kv / per_row,
                            (uint64_t)2 * num_blocks};
  const uint64_t strides[3] = {(uint64_t)n_kv * head_dim, row,
                               (uint64_t)kCachePage * n_kv * head_dim};
  const uint32_t box[4] = {(uint32_t)row, (uint32_t)kCachePage, (uint32_t)(cfg.hpc / per_row), 2};
  if (int rc = encode_tiled(&tmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(codes), dims,
                            strides, box,
                            row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B)) {
    return rc;
  }
  Decode8Params p;
  p.out = out;
  p.q = q;
  p.q_stride = q_row_stride;
  p.scales = scales;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.max_blocks = max_blocks_per_seq;
  p.num_seqs = num_seqs;
  p.n_kv = n_kv;
  p.G = n_q / n_kv;
  p.num_blocks = num_blocks;
  p.hpc = cfg.hpc;
  p.tg = cfg.tg;
  p.stages = cfg.stages;
  p.scale_log2 = scale * 1.4426950408889634f;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.group_counters = reinterpret_cast<int*>(ws);
  p.top_counters = p.group_counters + static_cast<size_t>(cfg.n_cta) * 2 * 2 * kParts8;
  p.part_lse = reinterpret_cast<float*>(ws + cfg.lse_at);
  p.part_o = reinterpret_cast<float*>(ws + cfg.o_at);
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool int8 = cache_format == VMPS_CACHE_INT8;
  if (dtype == VMPS_DTYPE_F16) {
    return int8 ? dispatch_decode8<__half, true>(head_dim, tmap, p, cfg, s)
                : dispatch_decode8<__half, false>(head_dim, tmap, p, cfg, s);
  }
  return int8 ? dispatch_decode8<__nv_bfloat16, true>(head_dim, tmap, p, cfg, s)
              : dispatch_decode8<__nv_bfloat16, false>(head_dim, tmap, p, cfg, s);
}

extern "C" int vmps_paged_decode_attention_cache8_args(const vmps_decode_cache8_args* a,
                                                       void* stream) {
  if (!a) return vmps::fail(VMPS_ERR_INVALID_ARG, "paged_decode_attention_cache8: NULL arguments");
  return vmps_paged_decode_attention_cache8(
      a->out, a->q, a->q_row_stride, a->codes, a->scales, a->block_tables, a->max_blocks_per_seq,
      a->seq_lens, a->num_seqs, a->n_q, a->n_kv, a->head_dim, a->block_size, a->num_blocks,
      a->scale, a->workspace, a->workspace_bytes, a->cache_format, a->dtype, stream);
}
