// Products with 4-bit weights and group scales, for a few activation rows:
//   Y[m][n] = sum_g scale[n][g] * sum_{k in g} X[m][k] * (code[n][k] - zero[n][g])
// optionally with the gated-MLP epilogue on a fused [gate; up] weight,
//   Y[m][i] = silu(gate[m][i]) * up[m][i].
//
// What bounds it.  Half a byte per weight and 2 M flops: the code stream from
// HBM is the bound for every M here.  At 6.5 TB/s an SM has to take in ~46
// codes a clock, so the work per code decides whether the stream is reached.
//
// Mathematics.  A code q is turned into the 16-bit float OFF + q by putting
// its four bits into the mantissa of a constant (OFF = 128 in bf16, 1024 in
// fp16: one and-or per two codes, exact).  With z the zero point and sx the
// group's sum of activations,
//   sum x (q - z) = sum x (OFF + q) - (OFF + z) sx,
// and the last term is what the group's fp32 accumulator starts from.  The
// matrix instruction (m16n8k16, codes as the 16-row side, activations as the
// 8-wide side) sums a group in fp32; the scale multiplies that sum in fp32,
// so neither scale nor zero point is ever rounded into a weight.
//
// The eight codes of a 32-bit word are taken in the order (0,4) (1,5) (2,6)
// (3,7): each pair is one mask of the word (shifted by 4 each time) and is one
// operand register.  The activations are stored in the same order in shared
// memory, so the sum over k is only reordered.  ldmatrix hands lane (g, c) the
// word c of row g's 32 codes, so two matrix instructions cover 32 adjacent
// codes and every group size (32, 64, 128) is a whole number of them.
//
// Work split.  A block of kRows = 16 or 32 output features (two 16-row tiles
// share each activation fragment from 9 rows on, where reading it from shared
// memory would otherwise be the bound) over all of K belongs to one CTA;
// contiguous equal shares of blocks go to one persistent CTA per SM.  A
// producer warp streams the codes with the tiled TMA (boxes of kRows rows x
// up to 16 chunks of 256 codes, 128-byte swizzle) into a ring; consumer
// warps take the chunks in turn; an epilogue warp adds their partial sums of a
// block in a fixed order, so no consumer waits for the adds and stores.
// Scales and zero points go straight to the registers of the lane quad that
// uses them, one chunk ahead.
//
// The activations of all rows must sit in shared memory.  Where M x K is too
// large, K is taken in phases (slices of whole chunks): a CTA runs a panel of
// its blocks through every phase and keeps the panel's sums in shared memory
// between them.  No partial sums leave the CTA.
//
// Launched with programmatic dependent launch: codes, scales and zero points
// do not depend on the kernel before, so the ring fills before the wait.
#include <mutex>

#include "vmps_abi_internal.h"
#include "vmps_common.cuh"

namespace vmps {
namespace {

constexpr int kW4MaxRows = 32;
// Consumer warps: a chunk is a chain of dependent steps, so four warps per
// scheduler where the registers allow it (one activation tile), else two.
__host__ __device__ constexpr int w4_consumers(int nt) { return nt == 1 ? 16 : 8; }
constexpr int w4_threads(int nt) { return 32 * (2 + w4_consumers(nt)); }  // + producer, epilogue
constexpr int kW4Chunk = 256;                        // codes of a row in a 128-byte line
constexpr int kW4MaxStages = 16;
constexpr int kW4SmemLimit = 226 * 1024;
constexpr int kW4Panel = 16;  // blocks a CTA carries through the phases at once
constexpr int kW4MaxRedSlots = 32;

struct W4Params {
  void* out;
  int64_t out_stride;
  const void* x;
  int64_t x_stride;
  const void* scales;
  const uint8_t* zeros;  // NULL: 8
  int M, N, K, ng;       // N: output features (half the weight's rows with silu)
  int silu;
  int chunks;            // of K (the last may be partial)
  int full_chunks;       // whole ones
  int cps;               // chunks per stage
  int slice;             // chunks per phase (a multiple of cps unless there is one phase)
  int phases;
  int stages;
  int team;              // consumer warps that share a block (a power of two)
  int red_slots;         // blocks whose partial sums can wait for the epilogue
  int blocks;            // of kRows features (per half with silu)
  int x_pitch;           // bytes between activation rows in shared memory
  int x_bytes, sx_bytes, red_bytes, acc_bytes, stage_bytes;
  int* err;
};

__device__ __forceinline__ void w4_pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void w4_pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void w4_tma_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0,
                                          int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

template <typename T> struct Code;
template <> struct Code<__nv_bfloat16> {
  static constexpr uint32_t kBits = 0x43004300u;  // 128, 128
  // 128 + z (z < 128) in fp32, by its mantissa bits.
  static __device__ __forceinline__ float offset_plus(uint32_t z) {
    return __uint_as_float(0x43000000u | (z << 16));
  }
};
template <> struct Code<__half> {
  static constexpr uint32_t kBits = 0x64006400u;  // 1024, 1024
  static __device__ __forceinline__ float offset_plus(uint32_t z) {
    return __uint_as_float(0x44800000u | (z << 13));
  }
};
// Codes (i, i + 4) of a word as OFF + code: one shift and one three-input
// logic operation, whose two constants have to be registers for that.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int i, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(word >> (4 * i)), "r"(mask), "r"(bits));
  return r;
}
// A wait that gives up, or finds that another has, leaves the CTA's abort flag
// set and returns: the roles then run to their ends on whatever is in shared
// memory, every access in bounds, no further wait lasting.
__device__ __forceinline__ void w4_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        int* err) {
  if (mbar_try_wait(bar, parity)) return;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return;
    if (clock64() - t0 > kWaitLimitCycles) {
      set_error(err, kDevErrTimeout);
      *abort_flag = 1;
      return;
    }
  }
}

// The order of a CTA's work, the same for all roles: panels of blocks, phases
// of a panel, blocks of the panel.  With silu a feature block is two blocks in
// a row, gate then up.
// A place in a ring of S slots and the parity of its current round.
struct RingPos {
  int at;
  uint32_t round;
  __device__ __forceinline__ void step(int n, int S) {
    at += n;
    while (at >= S) {
      at -= S;
      round ^= 1u;
    }
  }
};

template <typename T, int GROUP, int NT, int MT>
__global__ void __launch_bounds__(w4_threads(NT), 1)
    w4_kernel(const __grid_constant__ CUtensorMap map3, const __grid_constant__ CUtensorMap map2,
              const __grid_constant__ W4Params p) {
  constexpr int kRows = 16 * MT;
  constexpr int GP = kW4Chunk / GROUP;     // groups per chunk
  constexpr int UPG = GROUP / 32;          // 32-code units per group
  constexpr int NSZ = 2 * MT * GP / 4;     // (row, group) pairs a lane fetches per chunk
  constexpr int kFrag = MT * NT;
  constexpr int kConsumers = w4_consumers(NT);
  __shared__ uint64_t full_bar[kW4MaxStages];
  __shared__ uint64_t empty_bar[kW4MaxStages];
  __shared__ uint64_t red_full[kW4MaxRedSlots];
  __shared__ uint64_t red_empty[kW4MaxRedSlots];
  __shared__ volatile int s_abort;
  extern __shared__ __align__(1024) uint8_t smem[];

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // warp-uniform
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) set_error(p.err, kDevErrTimeout);
    return;
  }
  const int S = p.stages;
  uint8_t* ring = smem;
  uint8_t* xs = ring + S * p.stage_bytes;
  float* sx = reinterpret_cast<float*>(xs + p.x_bytes);
  float4* red = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(sx) + p.sx_bytes);
  float4* acc = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(red) + p.red_bytes);

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < S; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], p.team);
    }
    for (int i = 0; i < p.red_slots; ++i) {
      mbar_init(&red_full[i], p.team);
      mbar_init(&red_empty[i], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();

  const int halves = p.silu ? 2 : 1;
  const int G = gridDim.x;
  const int v0 = halves * static_cast<int>(static_cast<long long>(blockIdx.x) * p.blocks / G);
  const int v1 = halves * static_cast<int>(static_cast<long long>(blockIdx.x + 1) * p.blocks / G);
  const int panel = p.phases > 1 ? kW4Panel : (v1 - v0);
  const int wrows = halves * p.N;  // rows of the weight
  auto row_of = [&](int v) -> int {  // first weight row of block v
    return p.silu ? (v >> 1) * kRows + (v & 1) * p.N : v * kRows;
  };

  if (warp == 0) {
    // ── producer: codes only, so no PDL wait ─────────────────────────────────
    if (lane == 0) {
      prefetch_tmap(&map3);
      prefetch_tmap(&map2);
      RingPos rp = {0, 0u};
      int it = 0;
      for (int pv = v0; pv < v1 && !s_abort; pv += panel) {
        const int pe = min(pv + panel, v1);
        for (int ph = 0; ph < p.phases && !s_abort; ++ph) {
          const int c_end = min((ph + 1) * p.slice, p.chunks);
          for (int v = pv; v < pe && !s_abort; ++v) {
            for (int ch = ph * p.slice; ch < c_end; ch += p.cps, ++it, rp.step(1, S)) {
              const int st = rp.at;
              w4_wait(&empty_bar[st], rp.round ^ 1u, &s_abort, p.err);
              if (s_abort) break;
              uint8_t* dst = ring + st * p.stage_bytes;
              const int row = row_of(v);
              if (ch + p.cps <= p.full_chunks || p.full_chunks == p.chunks) {
                // Chunks past K read as zeros.
                mbar_arrive_expect_tx(&full_bar[st], p.cps * kRows * 128);
                tma_load_3d(dst, &map3, &full_bar[st], 0, row, ch);
              } else {
                // The stage with the row's partial last chunk: chunk by chunk,
                // each box cut off (zeros) at the row's end.
                const int n = min(p.cps, c_end - ch);
                mbar_arrive_expect_tx(&full_bar[st], n * kRows * 128);
                for (int i = 0; i < n; ++i) {
                  w4_tma_2d(dst + i * kRows * 128, &map2, &full_bar[st], (ch + i) * 128, row);
                }
              }
            }
          }
        }
      }
      // Every load in flight lands before the CTA exits.
      for (int j = max(0, it - S); j < it; ++j) mbar_wait(&full_bar[j % S], (j / S) & 1, p.err);
    }
    return;
  }

  if (warp == 1 + kConsumers) {
    // ── epilogue: adds the consumers' partial sums of each block ─────────────
    w4_pdl_wait();  // out may still be read by the previous kernel
    const int g = lane >> 2, c = lane & 3;
    T* out = static_cast<T*>(p.out);
    float gate[kFrag][4];
    RingPos rr = {0, 0u};
    for (int pv = v0; pv < v1; pv += panel) {
      const int pe = min(pv + panel, v1);
      for (int ph = 0; ph < p.phases; ++ph) {
        for (int v = pv; v < pe; ++v, rr.step(1, p.red_slots)) {
          const int slot = rr.at;
          w4_wait(&red_full[slot], rr.round, &s_abort, p.err);
          float4 sum[kFrag];
#pragma unroll
          for (int f = 0; f < kFrag; ++f) sum[f] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (ph > 0) {
#pragma unroll
            for (int f = 0; f < kFrag; ++f) sum[f] = acc[((v - pv) * kFrag + f) * 32 + lane];
          }
          for (int w = 0; w < p.team; ++w) {
#pragma unroll
            for (int f = 0; f < kFrag; ++f) {
              const float4 a = red[((slot * p.team + w) * kFrag + f) * 32 + lane];
              sum[f].x += a.x;
              sum[f].y += a.y;
              sum[f].z += a.z;
              sum[f].w += a.w;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&red_empty[slot]);
          if (ph + 1 < p.phases) {
#pragma unroll
            for (int f = 0; f < kFrag; ++f) acc[((v - pv) * kFrag + f) * 32 + lane] = sum[f];
            continue;
          }
          // Fragment: (feature g, row 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1).
          const bool up = p.silu && (v & 1);
#pragma unroll
          for (int f = 0; f < kFrag; ++f) {
            const float y[4] = {sum[f].x, sum[f].y, sum[f].z, sum[f].w};
            if (p.silu && !up) {
#pragma unroll
              for (int e = 0; e < 4; ++e) gate[f][e] = y[e];
              continue;
            }
            const int mt = f / NT, nt = f - mt * NT;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int feat = (p.silu ? v >> 1 : v) * kRows + mt * 16 + g + (e >> 1) * 8;
              const int m = nt * 8 + 2 * c + (e & 1);
              if (m >= p.M || feat >= p.N) continue;
              const float o = up ? gate[f][e] / (1.f + expf(-gate[f][e])) * y[e] : y[e];
              out[static_cast<int64_t>(m) * p.out_stride + feat] = Elt<T>::from_f(o);
            }
          }
        }
      }
    }
    return;
  }

  // ── consumers ──────────────────────────────────────────────────────────────
  const int w = (warp - 1) & (p.team - 1);       // place in the team
  const int team = (warp - 1) / p.team;          // takes blocks pv + team, + teams, ...
  const int teams = kConsumers / p.team;
  const int ctid = tid - 32;
  const int g = lane >> 2, c = lane & 3;
  const T* scales = static_cast<const T*>(p.scales);
  // The (row, group) pairs e = 4 i + c this lane fetches for its quad: group
  // e % GP of the chunk, row g + 8 * (e / GP) of the block; scale 0 past the
  // last group or row.  Nothing here uses a loaded value (that would wait).
  auto fetch = [&](int v, int ch, uint16_t (&sc)[NSZ], uint8_t (&zp)[NSZ]) {
    const int row0 = row_of(v) + g;
#pragma unroll
    for (int i = 0; i < NSZ; ++i) {
      const int e = 4 * i + c;
      const int grp = ch * GP + e % GP;
      const int row = row0 + 8 * (e / GP);
      sc[i] = 0;
      zp[i] = 8;
      if (grp < p.ng && row < wrows) {
        const uint32_t at = static_cast<uint32_t>(row) * p.ng + grp;  // < 2^31 (host check)
        sc[i] = reinterpret_cast<const uint16_t*>(scales)[at];
        if (p.zeros) zp[i] = p.zeros[at];
      }
    }
  };
  // ldmatrix rows of this lane: tiles (rows 0-7, unit u), (rows 8-15, u),
  // (rows 0-7, u + 1), (rows 8-15, u + 1) of a 16-row tile.
  const int mi = lane >> 3, r8 = lane & 7;
  const uint32_t a_lane = static_cast<uint32_t>((r8 + (mi & 1) * 8) * 128 + (((mi >> 1) ^ r8) << 4));
  const uint32_t ring_u32 = smem_u32(ring);
  uint32_t x_lane[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // Rows past M read row M - 1: their columns of the result are not used.
    x_lane[nt] = smem_u32(xs) + min(nt * 8 + g, p.M - 1) * p.x_pitch + c * 16;
  }
  uint32_t mask, bits;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask));
  asm volatile("mov.b32 %0, %1;" : "=r"(bits) : "n"(Code<T>::kBits));
  bool waited = false;
  RingPos rp = {0, 0u}, rr = {0, 0u};  // of the current panel and phase's first block
  for (int pv = v0; pv < v1; pv += panel) {
    const int pe = min(pv + panel, v1);
    for (int ph = 0; ph < p.phases; ++ph) {
      const int c_begin = ph * p.slice, c_end = min(c_begin + p.slice, p.chunks);
      const int nch = c_end - c_begin;
      // The chunks of the team's blocks are dealt to its warps in turn: `off` is
      // this warp's next one, counted from the current stage's first.
      const int spv = (nch + p.cps - 1) / p.cps;  // stages per block
      int off = w;
      int nv = pv + team, nc = w;  // block and chunk of the next one to fetch scales for
      uint16_t sc_next[NSZ];
      uint8_t zp_next[NSZ];
      auto advance = [&]() {
        while (nc >= nch) {
          nc -= nch;
          nv += teams;
        }
        if (nv < pe) fetch(nv, c_begin + nc, sc_next, zp_next);
      };
      advance();
      if (!waited) {
        w4_pdl_wait();  // X is the previous kernel's output
        waited = true;
      }
      if (p.phases > 1) named_barrier_sync(1, 32 * kConsumers);  // X of the last phase is done with
      {
        // Stage the slice of X: 8 values a thread, in the order (0 4 1 5 2 6 3
        // 7), and each group's sum.  A group is GROUP / 8 adjacent lanes.
        const int k0 = c_begin * kW4Chunk;
        const int units = nch * (kW4Chunk / 8);  // a multiple of 32
        for (int e = ctid; e < p.M * units; e += 32 * kConsumers) {
          const int m = e / units, u = e - m * units;
          const int k = k0 + u * 8;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (k < p.K) {
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + m * p.x_stride + k);
          }
          uint4 o;
          o.x = __byte_perm(v.x, v.z, 0x5410);
          o.y = __byte_perm(v.x, v.z, 0x7632);
          o.z = __byte_perm(v.y, v.w, 0x5410);
          o.w = __byte_perm(v.y, v.w, 0x7632);
          *reinterpret_cast<uint4*>(xs + m * p.x_pitch + u * 16) = o;
          const T* xv = reinterpret_cast<const T*>(&v);
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s += Elt<T>::to_f(xv[i]);
#pragma unroll
          for (int sh = 1; sh < GROUP / 8; sh <<= 1) s += __shfl_xor_sync(0xffffffffu, s, sh);
          if (u % (GROUP / 8) == 0) sx[(u / (GROUP / 8)) * (8 * NT) + m] = s;
        }
      }
      named_barrier_sync(1, 32 * kConsumers);
      if (pv == v0 && ph == 0) w4_pdl_trigger();

      RingPos cur = rp, red_at = rr;
      cur.step(team * spv, S);
      red_at.step(team, p.red_slots);
      for (int v = pv + team; v < pe; v += teams) {
        float total[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) total[mt][nt][e] = 0.f;
          }
        }
        for (int s0 = 0; s0 < nch; s0 += p.cps, cur.step(1, S)) {
          const int st = cur.at;
          w4_wait(&full_bar[st], cur.round, &s_abort, p.err);
          const int n_stage = min(p.cps, nch - s0);
          for (; off < n_stage; off += p.team) {
            uint32_t sz[NSZ];
#pragma unroll
            for (int i = 0; i < NSZ; ++i) sz[i] = sc_next[i] | (static_cast<uint32_t>(zp_next[i]) << 16);
            nc += p.team;
            advance();
            const int ch = s0 + off;  // chunk within the slice
            const uint32_t base = ring_u32 + st * p.stage_bytes + off * (kRows * 128) + a_lane;
            uint32_t a[MT][4][4];  // [unit pair][(row half) + 2 * (unit in pair)]
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                ldmatrix_x4(a[mt][u], (base ^ (u << 5)) + mt * 2048);  // 16-byte unit 2 u (+ 1), swizzled
              }
            }
#pragma unroll
            for (int gp = 0; gp < GP; ++gp) {
              float part[MT][NT][4];
              float sc[MT][2];
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int e = (mt * 2 + h) * GP + gp;
                  const uint32_t q = __shfl_sync(0xffffffffu, sz[e >> 2], (lane & ~3) | (e & 3));
                  const uint16_t sb = static_cast<uint16_t>(q);
                  sc[mt][h] = Elt<T>::to_f(*reinterpret_cast<const T*>(&sb));
                  const float zz = Code<T>::offset_plus(q >> 16);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    const float2 s2 = *reinterpret_cast<const float2*>(
                        sx + (ch * GP + gp) * (8 * NT) + nt * 8 + 2 * c);
                    part[mt][nt][2 * h] = -zz * s2.x;
                    part[mt][nt][2 * h + 1] = -zz * s2.y;
                  }
                }
              }
#pragma unroll
              for (int u = 0; u < UPG; ++u) {
                const int U = gp * UPG + u;
                uint4 xv[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                               : "=r"(xv[nt].x), "=r"(xv[nt].y), "=r"(xv[nt].z), "=r"(xv[nt].w)
                               : "r"(x_lane[nt] + (ch * 8 + U) * 64));
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const uint32_t lo = a[mt][U >> 1][(U & 1) * 2], hi = a[mt][U >> 1][(U & 1) * 2 + 1];
                  const uint32_t f0[4] = {code_pair(lo, 0, mask, bits), code_pair(hi, 0, mask, bits),
                                          code_pair(lo, 1, mask, bits), code_pair(hi, 1, mask, bits)};
                  const uint32_t f1[4] = {code_pair(lo, 2, mask, bits), code_pair(hi, 2, mask, bits),
                                          code_pair(lo, 3, mask, bits), code_pair(hi, 3, mask, bits)};
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    Mma<T>::run(part[mt][nt], f0, xv[nt].x, xv[nt].y);
                    Mma<T>::run(part[mt][nt], f1, xv[nt].z, xv[nt].w);
                  }
                }
              }
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    total[mt][nt][e] = fmaf(sc[mt][e >> 1], part[mt][nt][e], total[mt][nt][e]);
                  }
                }
              }
            }
          }
          off -= n_stage;
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty_bar[st]);
        }
        const int slot = red_at.at;
        w4_wait(&red_empty[slot], red_at.round ^ 1u, &s_abort, p.err);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            red[((slot * p.team + w) * kFrag + mt * NT + nt) * 32 + lane] =
                make_float4(total[mt][nt][0], total[mt][nt][1], total[mt][nt][2], total[mt][nt][3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_full[slot]);
        cur.step((teams - 1) * spv, S);
        red_at.step(teams, p.red_slots);
      }
      rp.step((pe - pv) * spv, S);
      rr.step(pe - pv, p.red_slots);
    }
  }
}

// ── host side ────────────────────────────────────────────────────────────────

int w4_nt(int M) { return M <= 8 ? 1 : (M <= 16 ? 2 : 4); }

// Shared-memory plan: the fewest phases whose activations leave the ring at
// least kW4MinRing bytes (an SM needs ~50 KB in flight to reach the stream).
constexpr int kW4MinRing = 56 * 1024;

bool w4_plan(W4Params* p, int group, int cta_blocks) {
  const int nt = w4_nt(p->M), mt = nt > 1 ? 2 : 1;
  const int rows = 16 * mt;
  const int line = rows * 128;  // bytes of one chunk of a block
  // A warp should take about four chunks of a block (its share of the block's
  // fixed costs), but all warps should have a block.
  const int cons = w4_consumers(nt);
  p->team = 1;
  while (p->team < cons && (p->team * 4 < p->chunks || p->team * cta_blocks < cons)) p->team *= 2;
  // Two blocks per team in flight to the epilogue (one with four activation
  // tiles, where a slot of a full team is 32 KB that the ring needs more).
  p->red_slots = cons / p->team * (nt > 2 ? 1 : 2);
  p->red_bytes = p->red_slots * p->team * mt * nt * 512;
  for (int phases = 1; phases <= 64; ++phases) {
    for (int cps = 16; cps >= 1; cps >>= 1) {
      if (cps * line > 32 * 1024 && cps > 1) continue;
      if (cps > 1 && cps / 2 >= p->chunks) continue;
      int slice = (p->chunks + phases - 1) / phases;
      if (phases > 1) slice = (slice + cps - 1) / cps * cps;
      p->x_pitch = slice * 512 + 64;  // 64 mod 128: rows g and g + 1 fill all banks
      p->x_bytes = (p->M * p->x_pitch + 127) / 128 * 128;
      p->sx_bytes = (slice * (kW4Chunk / group) * 8 * nt * 4 + 127) / 128 * 128;
      const int real_phases = (p->chunks + slice - 1) / slice;
      const int panel = cta_blocks < kW4Panel ? cta_blocks : kW4Panel;
      p->acc_bytes = real_phases > 1 ? panel * mt * nt * 512 : 0;
      const int left = kW4SmemLimit - p->x_bytes - p->sx_bytes - p->red_bytes - p->acc_bytes;
      p->stage_bytes = cps * line;
      int stages = left / p->stage_bytes;
      if (left < kW4MinRing || (stages < 4 && cps > 1)) continue;
      p->stages = stages < kW4MaxStages ? stages : kW4MaxStages;
      p->cps = cps;
      p->slice = slice;
      p->phases = real_phases;
      return true;
    }
  }
  return false;
}

template <typename T, int GROUP, int NT, int MT>
int w4_launch(const CUtensorMap& m3, const CUtensorMap& m2, const W4Params& p, int grid,
              cudaStream_t s) {
  static std::once_flag flags[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(VMPS_ERR_CUDA, "device index %d", dev);
  std::call_once(flags[dev], [] {
    cudaFuncSetAttribute(w4_kernel<T, GROUP, NT, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         kW4SmemLimit);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(w4_threads(NT));
  cfg.dynamicSmemBytes = static_cast<size_t>(p.stages) * p.stage_bytes + p.x_bytes + p.sx_bytes +
                         p.red_bytes + p.acc_bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, w4_kernel<T, GROUP, NT, MT>, m3, m2, p);
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "w4_gemm: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
}

template <typename T, int GROUP>
int w4_by_rows(const CUtensorMap& m3, const CUtensorMap& m2, const W4Params& p, int grid,
               cudaStream_t s) {
  switch (w4_nt(p.M)) {
    case 1: return w4_launch<T, GROUP, 1, 1>(m3, m2, p, grid, s);
    case 2: return w4_launch<T, GROUP, 2, 2>(m3, m2, p, grid, s);
    default: return w4_launch<T, GROUP, 4, 2>(m3, m2, p, grid, s);
  }
}

template <typename T>
int w4_by_group(int group, const CUtensorMap& m3, const CUtensorMap& m2, const W4Params& p,
                int grid, cudaStream_t s) {
  switch (group) {
    case 32: return w4_by_rows<T, 32>(m3, m2, p, grid, s);
    case 64: return w4_by_rows<T, 64>(m3, m2, p, grid, s);
    default: return w4_by_rows<T, 128>(m3, m2, p, grid, s);
  }
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" int vmps_w4_gemm_supported(int M, int N, int K, int group_size) {
  if (M < 0 || M > kW4MaxRows || N <= 0 || K <= 0) return 0;
  if (group_size != 32 && group_size != 64 && group_size != 128) return 0;
  return K % group_size == 0 ? 1 : 0;
}

extern "C" int vmps_w4_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                            const void* codes, const void* scales, const void* zeros, int M, int N,
                            int K, int group_size, int silu_mul, int dtype, void* stream) {
  const char* what = "w4_gemm";
  clear_error();
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (!vmps_w4_gemm_supported(M, N, K, group_size) ||
      2 * static_cast<int64_t>(N) * (K / group_size) > 0x7fffffff) {
    return fail(VMPS_ERR_UNSUPPORTED,
                "%s: M=%d N=%d K=%d group=%d (M <= %d, group 32, 64 or 128, K a multiple of it)",
                what, M, N, K, group_size, kW4MaxRows);
  }
  if (M == 0) return VMPS_OK;
  if (!out || !x || !codes || !scales) return fail(VMPS_ERR_INVALID_ARG, "%s: NULL pointer", what);
  if (x_row_stride < K || out_row_stride < N) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: row stride smaller than a row", what);
  }
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || (zeros && !aligned16(zeros)) ||
      (x_row_stride % 8) || (reinterpret_cast<uintptr_t>(out) & 1)) {
    return fail(VMPS_ERR_ALIGNMENT,
                "%s: x, codes, scales and zeros must be 16-byte aligned, x rows a multiple of 8 "
                "elements apart, out 2-byte aligned",
                what);
  }
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  int* err = nullptr;
  if (int rc = device_error_word(&err)) return rc;
  const int rows = w4_nt(M) > 1 ? 32 : 16;
  W4Params p;
  p.out = out;
  p.out_stride = out_row_stride;
  p.x = x;
  p.x_stride = x_row_stride;
  p.scales = scales;
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.M = M;
  p.N = N;
  p.K = K;
  p.ng = K / group_size;
  p.silu = silu_mul ? 1 : 0;
  p.chunks = (K + kW4Chunk - 1) / kW4Chunk;
  p.full_chunks = K / kW4Chunk;
  p.blocks = (N + rows - 1) / rows;
  p.err = err;
  const int grid = p.blocks < sms ? p.blocks : sms;
  if (!w4_plan(&p, group_size, (p.blocks + grid - 1) / grid * (p.silu ? 2 : 1))) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: no shared-memory plan for M=%d K=%d", what, M, K);
  }
  const uint64_t wrows = static_cast<uint64_t>(p.silu ? 2 : 1) * N;
  // Codes as {128 bytes, rows, whole chunks}: one box is a stage.  And as
  // {bytes, rows} for a partial last chunk.
  CUtensorMap m3, m2;
  {
    const uint64_t dims[2] = {(uint64_t)K / 2, wrows};
    const uint64_t strides[1] = {(uint64_t)K / 2};
    const uint32_t box[2] = {128, (uint32_t)rows};
    if (int rc = encode_tiled(&m2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims,
                              strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) {
      return rc;
    }
  }
  if (p.full_chunks > 0) {
    const uint64_t dims[3] = {128, wrows, (uint64_t)p.full_chunks};
    const uint64_t strides[2] = {(uint64_t)K / 2, 128};
    const uint32_t box[3] = {128, (uint32_t)rows, (uint32_t)p.cps};
    if (int rc = encode_tiled(&m3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims,
                              strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) {
      return rc;
    }
  } else {
    m3 = m2;  // never loaded through: every stage holds the partial chunk
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == VMPS_DTYPE_F16 ? w4_by_group<__half>(group_size, m3, m2, p, grid, s)
                                 : w4_by_group<__nv_bfloat16>(group_size, m3, m2, p, grid, s);
}
