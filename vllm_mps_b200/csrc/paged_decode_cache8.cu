// Kernel 11: decode attention over the 8-bit paged cache, one query token per
// sequence.
//
//   out[i][h] = softmax_t(scale * q[i][h] . K[t]) . V[t],  K, V = code * scale
//
// What bounds it: the codes' bytes from HBM (4 G operations per K and V code
// byte pair, G query heads a kv head).
//
//  * Work: tiles of 16 TG tokens of HPC kv heads, HPC * TG <= 8 consumer warps
//    (HPC: the largest divisor of n_kv up to 8; TG fills the CTA up to 8 warps
//    where there are few kv heads).  The tiles of all sequences are cut into equal
//    contiguous shares, one per CTA of a persistent grid (cache8_plan.h), so that
//    ragged batches and single long sequences both keep every SM streaming.
//  * A producer warp streams pages: a tiled TMA for the codes (K and V of HPC
//    heads, swizzled) and a bulk copy for their scales, into a ring of stages.
//  * A consumer warp takes 16 tokens of one kv head a stage.  The G query heads
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
//    rounding to fp16, relative to vref, a power of two that bounds V's scales so
//    far.  Weights are relative to 2^-11 of a running bound of the scores that is
//    raised when a score passes it by 2^4: they stay below 2^15, and what fp16
//    cannot hold of small ones is 2^-36 of the largest.  Sums of weights are
//    fp32 and unrounded.
//  * bf16 queries are scaled by a power of two per head, so that their largest
//    is in [2^13, 2^14), which fp16 holds as exactly as bf16 did but for values
//    below 2^-28 of it.
//  * A cut sequence: every piece leaves its normalised output and the logarithm
//    of its weights' sum in fp32 and arrives on a counter; the last to arrive
//    joins, in two rounds where there are many pieces.  Sums are in a fixed order:
//    results do not depend on who is last.
#include <mutex>
#include <utility>

#include "cache8.cuh"
#include "cache8_plan.h"
#include "vmps_abi_internal.h"

namespace vmps {
namespace {

constexpr int kMaxSeqs8 = 4096;
constexpr int kMaxKvHeads8 = 64;
constexpr int kMaxGroup8 = 16;
constexpr int kMaxStages8 = 8;
constexpr int kMaxWarps8 = 8;
constexpr int kThreads8 = 32 * (1 + kMaxWarps8);
// The workspace's counters; the records start where the 16-bit decode kernel's
// do, so that one workspace serves both.
constexpr size_t kCounterBytes8 = size_t(128) << 10;
constexpr size_t kRecordsAt8 = size_t(1) << 20;
constexpr float kLowest8 = -1e30f;  // the score bound of a piece that has seen nothing

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
  int* group_counters;  // [n_cta][2][hpc]
  int* top_counters;    // [n_cta][hpc]
  float* part_lse;      // [n_cta][2][hpc][NT][4][2]
  float* part_o;        // [n_cta][2][hpc][NT * D / 16][32 lanes][4]
  int* err;
};

// A published piece of a cut sequence: its run of CTAs, the sequence and its kv head, and
// how many arrivals were missing before its own (0: it was the last; lane 0 writes it).
struct Piece8 {
  int c0, c1, s, kvh, missing;
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

// Joins `count` records (every `step`-th CTA's from `cta` on, slot 1 in CTA c0, 0 in the
// others): the normalised output in o, the logarithm of the weights' sum in lse.
template <int D, int NT>
__device__ __forceinline__ void join_records(const Decode8Params& p, int cta, int step, int count,
                                             int c0, int h, int lane, float (&lse)[NT][2],
                                             float (&o)[NT][D / 16][4]) {
  constexpr int KS = D / 16;
  const int c = lane & 3;
  const float2* ml = reinterpret_cast<const float2*>(p.part_lse) + c;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) + lane;
  auto rec = [&](int k) {
    const int b = cta + k * step;
    return (static_cast<size_t>(b) * 2 + (b == c0 ? 1 : 0)) * p.hpc + h;
  };
  float top[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    top[nt][0] = top[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
  }
#pragma unroll 8
  for (int k = 0; k < count; ++k) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 v = __ldcg(ml + (rec(k) * NT + nt) * 4);
      top[nt][0] = fmaxf(top[nt][0], v.x);
      top[nt][1] = fmaxf(top[nt][1], v.y);
    }
  }
#pragma unroll 2
  for (int k = 0; k < count; ++k) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 v = __ldcg(ml + (rec(k) * NT + nt) * 4);
      const float w0 = fast_exp2(v.x - top[nt][0]), w1 = fast_exp2(v.y - top[nt][1]);
      sum[nt][0] += w0;
      sum[nt][1] += w1;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        const float4 x = __ldcg(po + ((rec(k) * NT + nt) * KS + mt) * 32);
        o[nt][mt][0] = fmaf(w0, x.x, o[nt][mt][0]);
        o[nt][mt][1] = fmaf(w1, x.y, o[nt][mt][1]);
        o[nt][mt][2] = fmaf(w0, x.z, o[nt][mt][2]);
        o[nt][mt][3] = fmaf(w1, x.w, o[nt][mt][3]);
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float r0 = 1.f / sum[nt][0], r1 = 1.f / sum[nt][1];
    lse[nt][0] = top[nt][0] + log2f(sum[nt][0]);
    lse[nt][1] = top[nt][1] + log2f(sum[nt][1]);
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      o[nt][mt][0] *= r0;
      o[nt][mt][1] *= r1;
      o[nt][mt][2] *= r0;
      o[nt][mt][3] *= r1;
    }
  }
}

// Output rows of a kv head from O^T fragments (rows g, g + 8 of m-tile mt: elements
// 16 mt + 2g and the next; columns 2c, 2c + 1: heads).
template <typename T, int D, int NT>
__device__ __forceinline__ void store_rows(T* rows, int G, int lane, const float (&f)[NT][2],
                                           const float (&o)[NT][D / 16][4]) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = nt * 8 + 2 * c + e;
      if (n >= G) continue;
      uint32_t* dst = reinterpret_cast<uint32_t*>(rows + n * D) + g;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        dst[mt * 8] = Elt<T>::pack(o[nt][mt][e] * f[nt][e], o[nt][mt][2 + e] * f[nt][e]);
      }
    }
  }
}

template <int D, int NT>
__device__ __forceinline__ void store_record(const Decode8Params& p, size_t rec, int lane,
                                             const float (&lse)[NT][2], const float (&f)[NT][2],
                                             const float (&o)[NT][D / 16][4]) {
  constexpr int KS = D / 16;
  float4* po = reinterpret_cast<float4*>(p.part_o) + rec * NT * KS * 32 + lane;
  float2* ml = reinterpret_cast<float2*>(p.part_lse) + rec * NT * 4;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      __stcg(po + (nt * KS + mt) * 32,
             make_float4(o[nt][mt][0] * f[nt][0], o[nt][mt][1] * f[nt][1],
                         o[nt][mt][2] * f[nt][0], o[nt][mt][3] * f[nt][1]));
    }
    if (lane < 4) __stcg(ml + nt * 4 + lane, make_float2(lse[nt][0], lse[nt][1]));
  }
}

// NT = 2 at head size 128 keeps 150 registers alive: one CTA per SM.
template <int D, int NT>
constexpr int kResident8 = (D == 128 && NT == 2) ? 1 : 2;

template <typename T, int D, int NT, bool kInt8>
__global__ void __launch_bounds__(kThreads8, kResident8<D, NT>)
decode8_kernel(const __grid_constant__ CUtensorMap tmap, const Decode8Params p) {
  constexpr int KS = D / 16;
  constexpr bool kF16 = std::is_same<T, __half>::value;
  __shared__ uint64_t full_bar[kMaxStages8];
  __shared__ uint64_t empty_bar[kMaxStages8];
  __shared__ volatile int s_abort;
  __shared__ int warp_sum[1 + kMaxWarps8];
  __shared__ Piece8 pieces_of[kMaxWarps8][2];
  extern __shared__ uint8_t dyn_smem[];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.num_seqs, hpc = p.hpc, TG = p.tg, stages = p.stages;
  const int page_bytes = 2 * hpc * kCachePage * D;
  const int stage_bytes = TG * page_bytes;
  const int scale_bytes = hpc * 2 * kCachePage * 4;  // of one page
  constexpr int kStateFloats = NT * (KS * 4 + 5);    // per lane: o, m, l, vref

  // [ring][scales][states that warps of one kv head hand over][prefix sums][lengths]
  const uint32_t base = smem_u32(dyn_smem);
  uint8_t* ring = dyn_smem + (((base + 1023u) & ~1023u) - base);
  float* ring_scales = reinterpret_cast<float*>(ring + stages * stage_bytes);
  float* states = ring_scales + stages * TG * scale_bytes / 4;
  int* wpref = reinterpret_cast<int*>(states + (TG / 2) * hpc * kStateFloats * 32);
  int* lens = wpref + n + 1;

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], hpc * TG);
    }
    fence_mbar_init();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ── lengths and the prefix sums of their weights ──────────────────────────
  const int tile_tokens = TG * kCachePage;
  {
    const int threads = blockDim.x;
    const int per = (n + threads - 1) / threads;
    for (int s = tid; s < n; s += threads) {
      int len = p.seq_lens[s];
      if (len <= 0) len = 0;
      if ((len + kCachePage - 1LL) / kCachePage > p.max_blocks) {
        if (blockIdx.x == 0) set_error(p.err, kDevErrSeqLen);
        len = p.max_blocks * kCachePage;
      }
      lens[s] = len;
    }
    __syncthreads();
    const int lo = min(n, tid * per), hi = min(n, lo + per);
    int sum = 0;
    for (int s = lo; s < hi; ++s) sum += c8_weight(c8_tiles(lens[s], tile_tokens));
    int incl = sum;
#pragma unroll
    for (int sh = 1; sh < 32; sh <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, sh);
      if (lane >= sh) incl += y;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += warp_sum[w];
    if (tid == 0) wpref[0] = 0;
    for (int s = lo; s < hi; ++s) {
      run += c8_weight(c8_tiles(lens[s], tile_tokens));
      wpref[s + 1] = run;
    }
    __syncthreads();
  }
  C8Shape sh;
  sh.num_seqs = n;
  sh.groups = p.n_kv / hpc;
  sh.n_cta = gridDim.x;
  sh.chunk = c8_chunk(wpref[n], sh.groups, sh.n_cta);
  const C8Pos begin = c8_pos(wpref, sh, static_cast<long long>(blockIdx.x) * sh.chunk);
  const C8Pos end = c8_pos(wpref, sh, static_cast<long long>(blockIdx.x + 1) * sh.chunk);
  C8Walk w;
  w.start(wpref, sh, begin, end);

  if (warp == 0) {
    // ── producer ────────────────────────────────────────────────────────────
    // Block-table entries are fetched 32 pages ahead of their use.
    if (lane == 0) prefetch_tmap(&tmap);
    int pg = 0, pg_end = 0;
    auto enter = [&]() {
      pg = w.j0 * TG;
      pg_end = min(w.j1 * TG, (lens[w.s] - 1) / kCachePage + 1);
    };
    auto fetch = [&](int& hg, int& count, int& phys) {
      count = 0;
      if (!w.valid) return;
      hg = w.hg;
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
    int hg, count, phys, hg2 = 0, count2, phys2 = 0;
    fetch(hg, count, phys);
    int stage = 0;
    uint32_t parity = 1;
    while (count > 0) {
      fetch(hg2, count2, phys2);
      const bool bad = phys < 0 || phys >= p.num_blocks;
      if (bad) set_error(p.err, kDevErrBlockRange);
      // Such a page's codes read as zeros (the tensor map's bounds), its scales as block 0's.
      const float* src = p.scales + (static_cast<size_t>(bad ? 0 : phys) * p.n_kv + hg * hpc) * 2 * kCachePage;
      if (bad) phys = p.num_blocks;
      for (int k = 0; k < count; k += TG) {
        const int np = min(TG, count - k);
        const bool ok = !s_abort && mbar_wait(&empty_bar[stage], parity, p.err);
        if (!__all_sync(0xffffffffu, ok)) {
          s_abort = 1;
          return;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[stage], np * (page_bytes + scale_bytes));
        __syncwarp();
        if (lane >= k && lane < k + np) {
          const int i = lane - k;
          tma_load_4d(ring + stage * stage_bytes + i * page_bytes, &tmap, &full_bar[stage], 0, 0,
                      hg * hpc, 2 * phys);
          bulk_load(ring_scales + (stage * TG + i) * (scale_bytes / 4), src, scale_bytes,
                    &full_bar[stage]);
        }
        if (++stage == stages) {
          stage = 0;
          parity ^= 1;
        }
      }
      hg = hg2;
      count = count2;
      phys = phys2;
    }
    return;
  }

  // ── consumers ─────────────────────────────────────────────────────────────
  const int cw = warp - 1;
  const int h = cw % hpc, tg = cw / hpc;
  const int g = lane >> 2, c = lane & 3;
  T* out = static_cast<T*>(p.out);
  const int n_q = p.n_kv * p.G;
  for (int s = blockIdx.x; s < n; s += gridDim.x) {  // rows of empty sequences
    if (lens[s] > 0) continue;
    uint4* o4 = reinterpret_cast<uint4*>(out + static_cast<int64_t>(s) * n_q * D);
    for (int e = tid - 32; e < n_q * D / 8; e += blockDim.x - 32) o4[e] = make_uint4(0u, 0u, 0u, 0u);
  }

  // This lane's ldmatrix row: token r (+ 8 for matrices 1 and 3), 16-byte chunk 2 kk (+ 1 for
  // matrices 2 and 3), at the place the tensor map's swizzle put it.
  uint32_t off[D / 32];
  {
    const int tok = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const int chunk = 2 * kk + (lane >> 4);
      const int at = D == 128 ? chunk ^ (tok & 7) : chunk ^ ((tok >> 1) & 3);
      off[kk] = tok * D + at * 16;
    }
  }
  const uint32_t k_base = smem_u32(ring) + tg * page_bytes + h * kCachePage * D;
  const uint32_t v_add = hpc * kCachePage * D;
  const float* my_scales = ring_scales + (tg * hpc + h) * 2 * kCachePage + g;

  Piece8* pend = pieces_of[cw];
  int n_pend = 0, n_arrived = 0, arrive_at = -1;
  // The counter a piece arrives on, and how many do.
  auto counter_of = [&](int i, int& members) -> int* {
    const int pieces = pend[i].c1 - pend[i].c0 + 1;
    const int size = c8_join_group(pieces);
    const int first = (static_cast<int>(blockIdx.x) - pend[i].c0) / size * size;
    members = min(size, pieces - first);
    const int lead = pend[i].c0 + first;
    return p.group_counters + (static_cast<size_t>(lead) * 2 + (first == 0 ? 1 : 0)) * hpc + h;
  };

  int stage = 0, it = 0;
  uint32_t parity = 0;
  for (; w.valid; w.next(wpref, sh, end)) {
    const int s = w.s, kvh = w.hg * hpc + h, len = lens[s];
    // Q^T as the B operand: k indices 2c, 2c+1 and 2c+8, 2c+9 of step ks are elements
    // 16 ks + 4c .. + 3 of head g.
    uint32_t qf[NT][KS][2];
    float fac[NT][2];  // of heads 2c, 2c + 1: score -> log2 units
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + g;
      const T* row = static_cast<const T*>(p.q) + s * p.q_stride +
                     (static_cast<int64_t>(kvh) * p.G + (head < p.G ? head : 0)) * D + 4 * c;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 16 * ks);
        qf[nt][ks][0] = head < p.G ? v.x : 0u;
        qf[nt][ks][1] = head < p.G ? v.y : 0u;
      }
      float mine = p.scale_log2;
      if constexpr (!kF16) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t x = qf[nt][ks][e];
            top = max(top, max((x << 16) & 0x7fffffffu, x & 0x7fff0000u));
          }
        }
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

    float m[NT][2], l[NT][2], o[NT][KS][4];  // m: the score bound less 11
    float vref = pow2(-126), vinv = pow2(126);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kLowest8;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }

    for (int j = w.j0; j < w.j1; ++j, ++it) {
      // After a wait that gave up, the rest runs through without waiting: the barriers
      // between warps still meet.
      if (!s_abort && !mbar_wait(&full_bar[stage], parity, p.err)) s_abort = 1;
      const int live = len - (j * TG + tg) * kCachePage;  // tokens from this page on
      if (live > 0) {
        const bool tail = live < kCachePage;
        const uint32_t kb = k_base + stage * stage_bytes;
        const float* sc = my_scales + stage * TG * (scale_bytes / 4);
        const float ks0 = sc[0], ks1 = sc[8];
        float vs0 = sc[16], vs1 = sc[24];
        // Two chains of products, so that they do not wait on each other.
        float x[NT][4], y[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
          y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
        }
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          uint32_t a[4];
          ldmatrix_x4(a, kb + off[kk]);
          uint32_t b[4], d[4];
          widen<kInt8, true>(a[0], b[0], b[2]);
          widen<kInt8, true>(a[1], b[1], b[3]);
          widen<kInt8, true>(a[2], d[0], d[2]);
          widen<kInt8, true>(a[3], d[1], d[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Mma<__half>::run(x[nt], b, qf[nt][2 * kk][0], qf[nt][2 * kk][1]);
            Mma<__half>::run(y[nt], d, qf[nt][2 * kk + 1][0], qf[nt][2 * kk + 1][1]);
          }
        }
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          x[nt][0] = (x[nt][0] + y[nt][0]) * fac[nt][0] * ks0;
          x[nt][1] = (x[nt][1] + y[nt][1]) * fac[nt][1] * ks0;
          x[nt][2] = (x[nt][2] + y[nt][2]) * fac[nt][0] * ks1;
          x[nt][3] = (x[nt][3] + y[nt][3]) * fac[nt][1] * ks1;
        }
        if (tail) {
          // Whatever the slots behind the length hold takes no part.
          if (g >= live) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = -INFINITY;
            vs0 = 0.f;
          }
          if (g + 8 >= live) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][2] = x[nt][3] = -INFINITY;
            vs1 = 0.f;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          raise |= fmaxf(x[nt][0], x[nt][2]) > m[nt][0] + 15.f;
          raise |= fmaxf(x[nt][1], x[nt][3]) > m[nt][1] + 15.f;
        }
        raise |= fmaxf(vs0, vs1) > vref;
        if (__any_sync(0xffffffffu, raise)) {
          float vm = fmaxf(vs0, vs1);
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, b));
          float down = 1.f;
          if (vm > vref && vm < INFINITY) {
            const int e = min(127, static_cast<int>(__float_as_uint(vm) >> 23) - 126);
            vref = pow2(e);
            down = vinv;  // old reference over the new one, below
            vinv = e < 127 ? pow2(-e) : __int_as_float(0x00400000);  // 2^-127
            down = vinv / down;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float m0 = fmaxf(x[nt][0], x[nt][2]), m1 = fmaxf(x[nt][1], x[nt][3]);
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) {
              m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, b));
              m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, b));
            }
            m0 = fmaxf(m[nt][0], m0 - 11.f);
            m1 = fmaxf(m[nt][1], m1 - 11.f);
            const float a0 = fast_exp2(m[nt][0] - m0), a1 = fast_exp2(m[nt][1] - m1);
            m[nt][0] = m0;
            m[nt][1] = m1;
            l[nt][0] *= a0;
            l[nt][1] *= a1;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
              o[nt][mt][0] *= a0 * down;
              o[nt][mt][1] *= a1 * down;
              o[nt][mt][2] *= a0 * down;
              o[nt][mt][3] *= a1 * down;
            }
          }
        }
        vs0 *= vinv;
        vs1 *= vinv;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float p0 = fast_exp2(x[nt][0] - m[nt][0]), p1 = fast_exp2(x[nt][1] - m[nt][1]);
          const float p2 = fast_exp2(x[nt][2] - m[nt][0]), p3 = fast_exp2(x[nt][3] - m[nt][1]);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          // C fragment (row = token, col = head) -> B fragment (k = token, n = head).
          pb[nt][0] = movmatrix_trans(Elt<__half>::pack(p0 * vs0, p1 * vs0));
          pb[nt][1] = movmatrix_trans(Elt<__half>::pack(p2 * vs1, p3 * vs1));
        }
        const uint32_t vb = kb + v_add;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          uint32_t a[4];
          ldmatrix_x4_trans(a, vb + off[kk]);
          if (!kInt8 && tail) {
            // e4m3 has NaN codes, and 0 * NaN is one: tokens 2c, 2c+1 and 2c+8, 2c+9.
            const uint32_t lo = (2 * c < live ? 0xffffu : 0u) | (2 * c + 1 < live ? 0xffff0000u : 0u);
            const uint32_t hi = (2 * c + 8 < live ? 0xffffu : 0u) | (2 * c + 9 < live ? 0xffff0000u : 0u);
            a[0] &= lo;
            a[1] &= hi;
            a[2] &= lo;
            a[3] &= hi;
          }
          uint32_t b[4], d[4];
          widen<kInt8, false>(a[0], b[0], b[1]);
          widen<kInt8, false>(a[1], b[2], b[3]);
          widen<kInt8, false>(a[2], d[0], d[1]);
          widen<kInt8, false>(a[3], d[2], d[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Mma<__half>::run(o[nt][2 * kk], b, pb[nt][0], pb[nt][1]);
            Mma<__half>::run(o[nt][2 * kk + 1], d, pb[nt][0], pb[nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[stage]);
      if (++stage == stages) {
        stage = 0;
        parity ^= 1;
      }
      if (n_arrived < n_pend && it >= arrive_at) {
        // A piece published two tiles ago: its stores are done, so the release is cheap.
        if (lane == 0) {
          int members;
          int* counter = counter_of(n_arrived, members);
          pend[n_arrived].missing = members - 1 - arrive_piece8(counter);
        }
        ++n_arrived;
      }
    }

#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) {
        l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], b);
        l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], b);
      }
    }
    // The warps of a kv head hand their states over, half of them to the other half each time.
    for (int half = TG / 2; half >= 1; half >>= 1) {
      float* slot = states + static_cast<size_t>(((tg & (half - 1)) * hpc + h) * kStateFloats) * 32 + lane;
      if (tg >= half && tg < 2 * half) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* z = slot + nt * (KS * 4 + 5) * 32;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) z[(mt * 4 + e) * 32] = o[nt][mt][e];
          }
          z[KS * 4 * 32] = m[nt][0];
          z[(KS * 4 + 1) * 32] = m[nt][1];
          z[(KS * 4 + 2) * 32] = l[nt][0];
          z[(KS * 4 + 3) * 32] = l[nt][1];
          z[(KS * 4 + 4) * 32] = vref;
        }
      }
      named_barrier_sync(1 + h, TG * 32);
      if (tg < half) {
        const float vr = slot[(KS * 4 + 4) * 32];
        const float v = fmaxf(vref, vr);
        const float va = vref / v, vb = vr / v;
        vref = v;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float* z = slot + nt * (KS * 4 + 5) * 32;
          const float n0 = z[KS * 4 * 32], n1 = z[(KS * 4 + 1) * 32];
          const float m0 = fmaxf(m[nt][0], n0), m1 = fmaxf(m[nt][1], n1);
          float a0 = fast_exp2(m[nt][0] - m0), a1 = fast_exp2(m[nt][1] - m1);
          float b0 = fast_exp2(n0 - m0), b1 = fast_exp2(n1 - m1);
          m[nt][0] = m0;
          m[nt][1] = m1;
          l[nt][0] = l[nt][0] * a0 + z[(KS * 4 + 2) * 32] * b0;
          l[nt][1] = l[nt][1] * a1 + z[(KS * 4 + 3) * 32] * b1;
          a0 *= va;
          a1 *= va;
          b0 *= vb;
          b1 *= vb;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            o[nt][mt][0] = o[nt][mt][0] * a0 + z[(mt * 4) * 32] * b0;
            o[nt][mt][1] = o[nt][mt][1] * a1 + z[(mt * 4 + 1) * 32] * b1;
            o[nt][mt][2] = o[nt][mt][2] * a0 + z[(mt * 4 + 2) * 32] * b0;
            o[nt][mt][3] = o[nt][mt][3] * a1 + z[(mt * 4 + 3) * 32] * b1;
          }
        }
      }
      named_barrier_sync(1 + h, TG * 32);
    }
    if (tg != 0) continue;

    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      f[nt][0] = vref / l[nt][0];
      f[nt][1] = vref / l[nt][1];
    }
    if (w.j0 == 0 && w.j1 == w.tiles) {
      store_rows<T, D, NT>(out + (static_cast<int64_t>(s) * n_q + kvh * p.G) * D, p.G, lane, f, o);
      continue;
    }
    if (n_pend == 2) {  // the plan leaves a CTA two pieces at most
      set_error(p.err, kDevErrSeqLen);
      continue;
    }
    const int c0 = c8_owner(wpref, sh, w.hg, s, 0);
    const int c1 = c8_owner(wpref, sh, w.hg, s, w.tiles - 1);
    const size_t rec = (static_cast<size_t>(blockIdx.x) * 2 + (static_cast<int>(blockIdx.x) == c0)) * hpc + h;
    float lse[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      lse[nt][0] = m[nt][0] + log2f(l[nt][0]);
      lse[nt][1] = m[nt][1] + log2f(l[nt][1]);
      // A piece whose weights are all zero (scores of -inf) adds nothing.
      if (l[nt][0] == 0.f) f[nt][0] = 0.f;
      if (l[nt][1] == 0.f) f[nt][1] = 0.f;
    }
    store_record<D, NT>(p, rec, lane, lse, f, o);
    if (lane == 0) pend[n_pend] = Piece8{c0, c1, s, kvh, -1};
    ++n_pend;
    arrive_at = it + 2;
  }

  // ── joining cut sequences ─────────────────────────────────────────────────
  __syncwarp();  // every lane's stores before lane 0's releases
  int last = 0;
  if (lane == 0) {
    for (int i = n_arrived; i < n_pend; ++i) {
      int members;
      int* counter = counter_of(i, members);
      pend[i].missing = members - 1 - arrive_piece8(counter);
    }
    for (int i = 0; i < n_pend; ++i) last |= (pend[i].missing == 0) << i;
  }
  last = __shfl_sync(0xffffffffu, last, 0);
  __syncwarp();  // every lane's loads after lane 0's acquire
  for (int i = 0; i < n_pend; ++i) {
    if (!(last & (1 << i))) continue;
    const int c0 = pend[i].c0, pieces = pend[i].c1 - c0 + 1;
    const int size = c8_join_group(pieces);
    const int first = (static_cast<int>(blockIdx.x) - c0) / size * size;
    float lse[NT][2], o[NT][KS][4], one[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) one[nt][0] = one[nt][1] = 1.f;
    int members;
    int* counter = counter_of(i, members);
    join_records<D, NT>(p, c0 + first, 1, members, c0, h, lane, lse, o);
    if (lane == 0) *counter = 0;
    if (size < pieces) {
      // Round two: this group's record takes the place of its first piece's.
      const int lead = c0 + first;
      store_record<D, NT>(p, (static_cast<size_t>(lead) * 2 + (first == 0)) * hpc + h, lane, lse,
                          one, o);
      __syncwarp();
      const int groups = (pieces + size - 1) / size;
      int* top = p.top_counters + static_cast<size_t>(c0) * hpc + h;
      int final_one = 0;
      if (lane == 0) final_one = arrive_piece8(top) == groups - 1;
      if (!__shfl_sync(0xffffffffu, final_one, 0)) continue;
      __syncwarp();
      join_records<D, NT>(p, c0, size, groups, c0, h, lane, lse, o);
      if (lane == 0) *top = 0;
    }
    store_rows<T, D, NT>(out + (static_cast<int64_t>(pend[i].s) * n_q + pend[i].kvh * p.G) * D, p.G,
                         lane, one, o);
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
Decode8Config configure8(int num_seqs, int n_q, int n_kv, int D, int sms) {
  Decode8Config cfg;
  cfg.hpc = kMaxWarps8;
  while (n_kv % cfg.hpc) --cfg.hpc;
  cfg.tg = 1;
  while (cfg.hpc * cfg.tg * 2 <= kMaxWarps8) cfg.tg *= 2;
  cfg.nt = n_q / n_kv > 8 ? 2 : 1;
  const int resident = (D == 128 && cfg.nt == 2) ? 1 : 2;
  cfg.n_cta = sms * resident;
  const size_t stage = static_cast<size_t>(cfg.tg) * cfg.hpc * (2 * kCachePage * D + 2 * kCachePage * 4);
  const size_t rest = 1024 + static_cast<size_t>(cfg.tg / 2) * cfg.hpc * cfg.nt * (D / 4 + 5) * 32 * 4 +
                      (2 * static_cast<size_t>(num_seqs) + 1) * 4;
  // Shared memory of an SM: 228 KB, 1 KB of it taken per CTA.
  const size_t room = resident == 1 ? 220u << 10 : 111u << 10;
  cfg.stages = kMaxStages8;
  while (cfg.stages > 2 && rest + cfg.stages * stage > room) --cfg.stages;
  cfg.smem = rest + cfg.stages * stage;
  const size_t recs = static_cast<size_t>(cfg.n_cta) * 2 * cfg.hpc;
  cfg.lse_at = kRecordsAt8;
  cfg.o_at = cfg.lse_at + align256_8(recs * cfg.nt * 8 * sizeof(float));
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
                         cudaFuncAttributeMaxDynamicSharedMemorySize, 226 << 10);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.n_cta);
  cfg.blockDim = dim3(32 * (1 + c.hpc * c.tg));
  cfg.dynamicSmemBytes = c.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, decode8_kernel<T, D, NT, kInt8>, tmap, p);
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
  return configure8(num_seqs, n_q, n_kv, head_dim, sms).workspace;
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
  if (!(scale > 0.f) || !(scale < 1e30f)) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: scale %g", what, (double)scale);
  }
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const Decode8Config cfg = configure8(num_seqs, n_q, n_kv, head_dim, sms);
  if (static_cast<size_t>(cfg.n_cta) * 3 * cfg.hpc * sizeof(int) > kCounterBytes8) {
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
  // The cache as {d, token, kv head, (block, K|V)}: the box [D][16][hpc][2] lands as
  // [K|V][head][token] rows of D bytes, their 16-byte chunks swizzled.
  CUtensorMap tmap;
  const uint64_t dims[4] = {(uint64_t)head_dim, (uint64_t)kCachePage, (uint64_t)n_kv,
                            (uint64_t)2 * num_blocks};
  const uint64_t strides[3] = {(uint64_t)n_kv * head_dim, (uint64_t)head_dim,
                               (uint64_t)kCachePage * n_kv * head_dim};
  const uint32_t box[4] = {(uint32_t)head_dim, (uint32_t)kCachePage, (uint32_t)cfg.hpc, 2};
  if (int rc = encode_tiled(&tmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(codes), dims,
                            strides, box,
                            head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B)) {
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
  p.top_counters = p.group_counters + static_cast<size_t>(cfg.n_cta) * 2 * cfg.hpc;
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
