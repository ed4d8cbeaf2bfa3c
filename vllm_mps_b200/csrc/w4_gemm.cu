// Products with 4-bit weights and group scales, for a few activation rows:
//   Y[m][n] = sum_g scale[n][g] * sum_{k in g} X[m][k] * (code[n][k] - zero[n][g])
// optionally with the gated-MLP epilogue on a fused [gate; up] weight,
//   Y[m][i] = silu(gate[m][i]) * up[m][i].
//
// What bounds it.  Half a byte per weight and 2 M flops: the code stream from
// HBM is the bound for every M here.  At 6.5 TB/s an SM has to take in ~46
// codes a clock, so the work per code decides whether the stream is reached:
// it is not quite (about 290 instructions per 4096 codes, half the issue slots
// used).  Measured, bf16, groups of 128: 128256 x 4096 at 16 rows 68 us (4.0
// TB/s), [gate; up] 2 x 14336 x 4096 at one row 18.3 us (3.4 TB/s), of which 4 us
// are the launch and the activations; 4096 x 14336 at 5 rows, groups of 64,
// 20.5 us (1.6 TB/s: its activations are staged in two phases, 4 us each).  Above
// 16 rows, with 2 to 5 phases and a fragment read per block, it is far from the
// stream: 128256 x 4096 takes 135 us at 24 rows, 179 at 32.
//
// Mathematics.  A code q becomes the fp16 number OFF + q by putting its four
// bits into the mantissa of a constant (1024 where they land in bits 0-3 of a
// half, 64 in bits 4-7; exact), one and-or per two codes.  With z the zero
// point,
//   sum x (q - z) = sum x (OFF + q) - sum x OFF - z sum x,
// where the last two sums depend on the activations alone (computed once per
// CTA) and are what the group's fp32 accumulator starts from.  The matrix
// instruction (m16n8k16, codes as the 16-row side, activations as the 8-wide
// side) sums a group in fp32; the scale multiplies that sum in fp32, so
// neither scale nor zero point is ever rounded into a weight.  What the offset
// costs is fp32 bits of that sum: measured (fp16, K 4096) 0.012 x 2^-12 of
// sum |x| scale at most for activations of random sign, 0.76 x 2^-12 where all
// are near 30.  Rounding a weight to four bits costs such a sum some 25 times as
// much, and taking half of the offset off after the products instead (0.24 x
// 2^-12) 2 to 5 % of the time.
//
// bf16 activations go through the same fp16 instruction: each group of a row
// is multiplied by the power of two that brings its largest magnitude into
// [2^14, 2^15), which its fp32 sum is divided by again.  A bf16 significand
// fits fp16's; only values below 2^-29 of the group's largest lose bits (less
// than 2^-39 of it).  bf16's own mantissa holds the four bits in one place
// only, which costs seven operations per word instead of five.
//
// A row with an infinity or NaN would come out as NaN throughout, the offsets'
// share being taken off as inf - inf.  Such values decide the whole sum, so where
// the staging meets one the epilogue sums them alone, from the definition.
//
// The eight codes of a 32-bit word are taken in the order (0,4) (1,5) (2,6)
// (3,7): each pair is one mask of the word or of the word shifted by 8, and is
// one operand register.  The activations are stored in the same order in
// shared memory, so the sum over k is only reordered.  ldmatrix hands lane
// (g, c) the word c of row g's 32 codes, so two matrix instructions cover 32
// adjacent codes and every group size (32, 64, 128) is a whole number of them.
//
// Work split.  A block of kRows = 16 output features (32 for 9 to 16 activation
// rows: two 16-row tiles then share each activation fragment, whose reads from
// shared memory would otherwise be the bound; above 16 rows their accumulators
// do not fit the registers) over all of K belongs to one CTA;
// contiguous equal shares of blocks go to one persistent CTA per SM.  The
// warps form teams; a team takes every teams-th block, its warps the block's
// chunks (2 or 4 KB of codes) in turn, and adds their partial sums of the block
// through shared memory in a fixed order.  Every warp streams its own chunks
// with 16-byte asynchronous copies into a private pair of slots, so nothing but
// the block's sum is waited for by more than one warp; 32 or 64 KB are in
// flight.  (With one bulk copy per row or one tensor box per block the copy
// engine's cost per line capped the stream at 60 % of this.)  Scales and zero points go
// straight to the registers of the lane quad that uses them, as many chunks
// ahead as the codes.
//
// The activations of all rows must sit in shared memory.  Where M x K is too
// large, K is taken in phases (slices of whole chunks): a CTA runs a panel of
// its blocks through every phase and keeps the panel's sums in shared memory
// between them.  No partial sums leave the CTA.
//
// Launched with programmatic dependent launch (the prologue overlaps the end of
// the kernel before; everything is read after its wait).
#include <mutex>
#include <type_traits>

#include "vmps_abi_internal.h"
#include "vmps_common.cuh"
#include "w4_plan.h"

namespace vmps {
namespace {

struct W4Params : W4Plan {
  void* out;
  int64_t out_stride;
  const void* x;
  int64_t x_stride;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;  // NULL: 8
  int M, N, K, ng;       // N: output features (half the weight's rows with silu)
  int silu;
  int blocks;            // of kRows features (per half with silu)
};

__device__ __forceinline__ void w4_pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void w4_pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void w4_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void w4_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void w4_wait_pending() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// (a & mask) | bits: one three-input operation, whose two constants have to be
// registers for that.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}

// A scale (low half) and a zero point packed for one shuffle, and back.  The
// zero point travels as a number of the scale's type (exact for 8 bits).
template <typename T> struct ScaleZero;
template <> struct ScaleZero<__half> {
  static __device__ __forceinline__ uint32_t pack(uint32_t scale, uint32_t zero) {
    const __half z = __hsub(__ushort_as_half(static_cast<unsigned short>(0x6400u | zero)),
                            __ushort_as_half(0x6400));
    return scale | (static_cast<uint32_t>(__half_as_ushort(z)) << 16);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float& scale, float& zero) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    scale = f.x;
    zero = f.y;
  }
};
template <> struct ScaleZero<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(uint32_t scale, uint32_t zero) {
    const float z = __uint_as_float(0x4B000000u | zero) - 8388608.f;  // exact
    return scale | (__float_as_uint(z) & 0xFFFF0000u);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float& scale, float& zero) {
    scale = __uint_as_float(w << 16);
    zero = __uint_as_float(w & 0xFFFF0000u);
  }
};

// The instruction of Mma<__half> with the sums' start in registers of its own.
__device__ __forceinline__ void w4_mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                            float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// What row m's infinities and NaN make of weight row n's sum, or y if it has none.
template <typename T, int GROUP>
__device__ __forceinline__ float w4_nonfinite(const W4Params& p, int n, int m, float y) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  const uint4* row = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + m * p.x_stride);
  const uint8_t* codes = p.codes + static_cast<int64_t>(n) * (p.K / 2);
  bool found = false;
  float sum = 0.f;
#pragma unroll 1
  for (int k8 = 0; k8 < p.K / 8; ++k8) {
    const uint4 v = row[k8];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
      if ((bits & kExp) == kExp) {
        const int k = k8 * 8 + i;
        const int64_t at = static_cast<int64_t>(n) * p.ng + k / GROUP;
        const int q = (codes[k >> 1] >> (4 * (k & 1))) & 15;
        const int z = p.zeros ? p.zeros[at] : 8;
        const unsigned short half = static_cast<unsigned short>(bits);
        const float x = Elt<T>::to_f(*reinterpret_cast<const T*>(&half));
        found = true;
        sum += Elt<T>::to_f(static_cast<const T*>(p.scales)[at]) * (x * static_cast<float>(q - z));
      }
    }
  }
  return found ? sum : y;
}

// The same for a fragment's four values: (feature feat, row m), (feat, m + 1),
// (feat + 8, m), (feat + 8, m + 1), of the weight's second half with `up`.  Only
// ever runs after the staging met such a value.
template <typename T, int GROUP>
__device__ __noinline__ float4 w4_nonfinite4(const W4Params& p, int feat, int m, bool up, float4 y) {
  float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int n = feat + (e >> 1) * 8, r = m + (e & 1);
    if (n < p.N && r < p.M) v[e] = w4_nonfinite<T, GROUP>(p, n + (up ? p.N : 0), r, v[e]);
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// ZP: with zero points.  Without, every row's sum of a group starts from the
// same numbers: 128256 x 4096 at 16 rows takes 73.4 us so, 75.0 with the 8 as
// a zero point of every group.
template <typename T, int GROUP, int NT, int MT, bool ZP>
__global__ void __launch_bounds__(kW4Threads, 1) w4_kernel(const __grid_constant__ W4Params p) {
  constexpr int kRows = 16 * MT;
  constexpr int kW4ChunkBytes = w4_chunk_bytes(NT);
  constexpr int kCodes = kW4ChunkBytes * 2 / kRows;  // codes of a row in a chunk
  constexpr int kRowBytes = kCodes / 2;
  constexpr int kUnits = kRowBytes / 16;             // 32-code units of a row
  constexpr int GP = kCodes / GROUP;                 // groups per chunk
  constexpr int UPG = GROUP / 32;
  constexpr int NSZ = (2 * MT * GP + 3) / 4;         // (row, group) pairs a lane fetches per chunk
  constexpr int kFrag = MT * NT;
  constexpr bool kScaled = !std::is_same<T, __half>::value;
  constexpr int kPlanes = w4_planes(kScaled, ZP);
  // Shared memory: rings | activations | group sums | partial sums | gate sums
  // (silu) | panel sums (several phases).
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t s_free[kW4Warps];  // free ring slots that hold partial sums
  static_assert(kFrag * 512 <= kW4ChunkBytes, "a block's sums fit a ring slot");

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // warp-uniform
  const int T_ = p.team;
  const int teams = kW4Warps / T_;
  const int w = warp & (T_ - 1);  // place in the team
  const int team = warp / T_;     // takes blocks pv + team, + teams, ...
  uint8_t* xs = smem + kW4Warps * kW4Depth * kW4ChunkBytes;
  // [group][plane][row]; see w4_planes.
  float* sx = reinterpret_cast<float*>(xs + p.x_bytes);
  float* red = sx + p.sx_bytes / 4 + team * T_ * kFrag * 128;  // the team's (first buffer)
  constexpr int kRedFloats = kW4Warps * kFrag * 128;           // of a buffer, all teams
  constexpr int kRedBufs = w4_red_bufs(NT);
  float* gate = sx + p.sx_bytes / 4 + kRedBufs * kRedFloats + team * kFrag * 128;  // with silu
  float* acc = sx + p.sx_bytes / 4 + kRedBufs * kRedFloats + (p.silu ? teams : 0) * kFrag * 128;

  const int halves = p.silu ? 2 : 1;
  const int G = gridDim.x;
  const int v0 = halves * static_cast<int>(static_cast<long long>(blockIdx.x) * p.blocks / G);
  const int v1 = halves * static_cast<int>(static_cast<long long>(blockIdx.x + 1) * p.blocks / G);
  const int wrows = halves * p.N;  // rows of the weight
  const uint32_t row_bytes = static_cast<uint32_t>(p.K) / 2;
  // First weight row of block v.  With silu a feature block is two blocks in a
  // row, gate then up, both of one team.
  auto row_of = [&](int v) -> int {
    return p.silu ? (v >> 1) * kRows + (v & 1) * p.N : v * kRows;
  };
  // Teams take feature blocks: `halves` adjacent blocks of every halves * teams.
  const int stride = halves * teams;
  auto next_block = [&](int v) -> int {
    return p.silu && !(v & 1) ? v + 1 : v + stride - (halves - 1);
  };

  // ── the stream: this warp's chunks in the order it will take them ──────────
  // (panel, phase, block, chunk); dealing starts at w in every phase.
  const uint32_t ring = smem_u32(smem) + warp * kW4Depth * kW4ChunkBytes;
  // A copy instruction takes 64 bytes of eight rows (whole sectors); the 16-byte
  // units of a row are swizzled so that ldmatrix's eight rows never share a
  // bank.  Copies of one row differ in the unit's bits 2 and up, untouched by
  // the lane's own, so their targets differ by an exclusive or.
  constexpr int kCols = kRowBytes / 64, kRowSets = kRows / 8;
  auto swz = [](int row, int unit) -> int {  // two rows share 128 bytes where a row has 64
    return unit ^ (kUnits == 4 ? (row >> 1) & 3 : row & 7);
  };
  const int g = lane >> 2, c = lane & 3;
  const uint32_t l_dst = g * kRowBytes + swz(g, c) * 16;
  // (row, group) pairs e = 4 i + c of this lane's quad: group e % GP of the
  // chunk, row g + 8 * (e / GP) of the block.
  const uint32_t end_of_ring = ring + kW4Depth * kW4ChunkBytes;
  int s_pv = v0, s_ph = 0, s_v = v0 + halves * team, s_c = w;
  int s_nch = min(p.slice, p.chunks);  // of the phase
  bool s_on = true, s_rows_full = false;
  uint32_t s_dst = ring;
  const uint8_t* s_src = nullptr;  // this lane's first 16 bytes of the next chunk
  uint32_t s_at = 0;               // its first (row, group) pair
  auto settle = [&]() {  // to the next chunk that exists
    for (;;) {
      const int pe = min(s_pv + p.panel, v1);
      while (s_c >= s_nch && s_v < pe) {
        s_c -= s_nch;
        s_v = next_block(s_v);
      }
      if (s_v < pe) break;
      if (++s_ph == p.phases) {
        s_ph = 0;
        s_pv += p.panel;
        if (s_pv >= v1) {
          s_on = false;
          return;
        }
      }
      s_nch = min(p.slice, p.chunks - s_ph * p.slice);
      s_v = s_pv + halves * team;
      s_c = w;
    }
    const int ch = s_ph * p.slice + s_c, row0 = row_of(s_v);
    s_rows_full = row0 + kRows <= wrows;
    s_src = p.codes + static_cast<uint64_t>(static_cast<uint32_t>(row0 + g)) * row_bytes +
            (ch * kRowBytes + c * 16);
    s_at = static_cast<uint32_t>(row0 + g + 8 * (c / GP)) * p.ng + ch * GP + c % GP;
  };
  uint16_t sc_next[NSZ];
  uint8_t zp_next[NSZ];
  // Starts the stream's next chunk: its codes into the next ring slot, this
  // lane's scales and zero points into registers.  Nothing here uses a loaded
  // value (that would wait for it).
  auto start_next = [&]() {
    if (s_on) {
      const uint16_t* scales = static_cast<const uint16_t*>(p.scales);
      const int ch = s_ph * p.slice + s_c;
      if (s_rows_full && (ch + 1) * kCodes <= p.K) {
#pragma unroll
        for (int r = 0; r < kRowSets; ++r) {
          const uint8_t* src = s_src + static_cast<uint64_t>(row_bytes) * (8 * r);
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            w4_copy16((s_dst + (l_dst ^ (i << 6))) + r * 8 * kRowBytes, src + i * 64);
          }
        }
#pragma unroll
        for (int i = 0; i < NSZ; ++i) {
          const uint32_t j = s_at + (4 * i) % GP + 8 * (4 * i / GP) * p.ng;
          if (2 * MT * GP >= 4 || c < 2 * MT * GP) sc_next[i] = scales[j];
          if (ZP && (2 * MT * GP >= 4 || c < 2 * MT * GP)) zp_next[i] = p.zeros[j];
        }
      } else {
        // The weight's last rows or a row's last codes: only what exists, and
        // scale 0 for the rest (what the slot holds there is finite).
        const int row0 = row_of(s_v);
#pragma unroll
        for (int r = 0; r < kRowSets; ++r) {
          const uint8_t* src = s_src + static_cast<uint64_t>(row_bytes) * (8 * r);
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            if (static_cast<uint32_t>(ch) * kRowBytes + i * 64 + c * 16 < row_bytes &&
                row0 + g + 8 * r < wrows) {
              w4_copy16((s_dst + (l_dst ^ (i << 6))) + r * 8 * kRowBytes, src + i * 64);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NSZ; ++i) {
          const int e = 4 * i + c;
          sc_next[i] = 0;
          zp_next[i] = 8;  // any that is finite
          if (ch * GP + e % GP < p.ng && row0 + g + 8 * (e / GP) < wrows && e < 2 * MT * GP) {
            const uint32_t j = s_at + (4 * i) % GP + 8 * (4 * i / GP) * p.ng;
            sc_next[i] = scales[j];
            if (ZP) zp_next[i] = p.zeros[j];
          }
        }
      }
      s_c += T_;
      if (s_c < s_nch) {
        s_src += T_ * kRowBytes;
        s_at += T_ * GP;
      } else {
        settle();
      }
    }
    w4_commit();
    s_dst += kW4ChunkBytes;
    if (s_dst == end_of_ring) s_dst = ring;
  };
  settle();
  // Nothing is read before the kernels ahead are done: X is theirs, and the
  // codes may be (a weight that was only just quantised).  The next launch's
  // CTAs find no room beside this one's, so an early stream would gain nothing.
  w4_pdl_wait();
  start_next();

  // ── the products ───────────────────────────────────────────────────────────
  const int mi = lane >> 3, r8 = lane & 7;
  // ldmatrix rows of this lane: tiles (rows 0-7, unit u), (rows 8-15, u),
  // (rows 0-7, u + 1), (rows 8-15, u + 1) of a 16-row tile; u is even.
  const int a_row = r8 + (mi & 1) * 8;
  const uint32_t a_lane = static_cast<uint32_t>(a_row * kRowBytes + swz(a_row, mi >> 1) * 16);
  uint32_t x_lane[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // Rows past M read row M - 1: their columns of the result are not used.
    x_lane[nt] = smem_u32(xs) + min(nt * 8 + g, p.M - 1) * p.x_pitch + c * 16;
  }
  uint32_t mask_lo, mask_hi, bits_lo, bits_hi;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask_lo));
  asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(mask_hi));
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(bits_lo));  // 1024, 1024
  asm volatile("mov.b32 %0, 0x54005400;" : "=r"(bits_hi));  // 64, 64
  float total[MT][NT][4];
  uint32_t r_src = ring;  // the next chunk's ring slot

  // One chunk: chunk `ch` of the slice, from the next ring slot.
  auto chunk = [&](int ch) {
    w4_wait_pending<0>();
    __syncwarp();  // every lane's copies have landed, and the last chunk is read
    uint32_t sz[NSZ];
#pragma unroll
    for (int i = 0; i < NSZ; ++i) sz[i] = ZP ? ScaleZero<T>::pack(sc_next[i], zp_next[i]) : sc_next[i];
    start_next();
    const uint32_t base = r_src + a_lane;
    r_src += kW4ChunkBytes;
    if (r_src == end_of_ring) r_src = ring;
    const uint32_t x_chunk = ch * (kUnits * 64);
    const float* s_chunk = sx + ch * (GP * kPlanes * 8 * NT) + 2 * c;
    uint32_t a[MT][4];  // a pair of units: [(row half) + 2 * (unit in pair)]
#pragma unroll
    for (int gp = 0; gp < GP; ++gp) {
      float part[MT][NT][4], start[MT][NT][4];
      float sc[MT][2];
      const float* sg = s_chunk + gp * (kPlanes * 8 * NT);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = (mt * 2 + h) * GP + gp;
          const uint32_t q = __shfl_sync(0xffffffffu, sz[e >> 2], (lane & ~3) | (e & 3));
          float zero;
          ScaleZero<T>::unpack(q, sc[mt][h], zero);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 off2 = *reinterpret_cast<const float2*>(sg + nt * 8);
            start[mt][nt][2 * h] = off2.x;
            start[mt][nt][2 * h + 1] = off2.y;
            if (ZP) {
              const float2 sum2 = *reinterpret_cast<const float2*>(sg + 8 * NT + nt * 8);
              start[mt][nt][2 * h] = fmaf(-zero, sum2.x, off2.x);
              start[mt][nt][2 * h + 1] = fmaf(-zero, sum2.y, off2.y);
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UPG; ++u) {
        const int U = gp * UPG + u;
        if ((U & 1) == 0) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            ldmatrix_x4(a[mt], (base ^ (U << 4)) + mt * 16 * kRowBytes);  // units U, U + 1
          }
        }
        uint4 xv[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(xv[nt].x), "=r"(xv[nt].y), "=r"(xv[nt].z), "=r"(xv[nt].w)
                       : "r"(x_lane[nt] + x_chunk + U * 64));
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint32_t lo = a[mt][(U & 1) * 2], hi = a[mt][(U & 1) * 2 + 1];
          const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
          const uint32_t f0[4] = {and_or(lo, mask_lo, bits_lo), and_or(hi, mask_lo, bits_lo),
                                  and_or(lo, mask_hi, bits_hi), and_or(hi, mask_hi, bits_hi)};
          const uint32_t f1[4] = {and_or(lo8, mask_lo, bits_lo), and_or(hi8, mask_lo, bits_lo),
                                  and_or(lo8, mask_hi, bits_hi), and_or(hi8, mask_hi, bits_hi)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (u == 0) {
              const float* from = start[mt][nt];
              w4_mma_from(part[mt][nt], f0, xv[nt].x, xv[nt].y, from[0], from[1], from[2], from[3]);
            } else {
              Mma<__half>::run(part[mt][nt], f0, xv[nt].x, xv[nt].y);
            }
            Mma<__half>::run(part[mt][nt], f1, xv[nt].z, xv[nt].w);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float2 down = make_float2(1.f, 1.f);
        if (kScaled) down = *reinterpret_cast<const float2*>(sg + (kPlanes - 1) * 8 * NT + nt * 8);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = kScaled ? part[mt][nt][e] * ((e & 1) ? down.y : down.x) : part[mt][nt][e];
            total[mt][nt][e] = fmaf(sc[mt][e >> 1], y, total[mt][nt][e]);
          }
        }
      }
    }
  };
  auto team_sync = [&]() {
    if (T_ == 1) {
      __syncwarp();
    } else {
      named_barrier_sync(1 + team, 32 * T_);
    }
  };

  T* out = static_cast<T*>(p.out);
  int red_buf = 0, turn = 0;
  int nonfinite = 0;  // an activation is (the same for all threads)
  for (int pv = v0; pv < v1; pv += p.panel) {
    const int pe = min(pv + p.panel, v1);
    for (int ph = 0; ph < p.phases; ++ph) {
      const int nch = min(p.slice, p.chunks - ph * p.slice);
      if (p.phases > 1) __syncthreads();  // the last phase's X is done with
      int met = 0;
      {
        // Stage the slice of X, in the order (0 4 1 5 2 6 3 7), and each group's
        // sums.  GROUP / 32 adjacent lanes take a row's group, 32 values each: one
        // maximum and sum across lanes per 32 values (16 rows x 4096 took 5 us
        // longer with one per 8).
        constexpr int kLanes = GROUP / 32, kAtOnce = kW4Threads / kLanes;
        const int groups = nch * GP, g0 = ph * p.slice * GP;
        const int t = tid % kLanes;
        int m = tid / kLanes / groups, gr = tid / kLanes - m * groups;
        const int step_m = kAtOnce / groups, step_g = kAtOnce - step_m * groups;
        while (__any_sync(0xffffffffu, m < p.M)) {
          const bool on = m < p.M;
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = make_uint4(0u, 0u, 0u, 0u);
          if (on && g0 + gr < p.ng) {
            const uint4* src = reinterpret_cast<const uint4*>(
                static_cast<const T*>(p.x) + m * p.x_stride + (g0 + gr) * GROUP + t * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = src[j * kLanes];
          }
          float up = 1.f;
          if (kScaled) {
            // Bit patterns of magnitudes order as integers, NaN above all.
            uint32_t top2 = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              top2 = __vmaxu2(__vmaxu2(top2, v[j].x & 0x7FFF7FFFu), v[j].y & 0x7FFF7FFFu);
              top2 = __vmaxu2(__vmaxu2(top2, v[j].z & 0x7FFF7FFFu), v[j].w & 0x7FFF7FFFu);
            }
            uint32_t top = max(top2 >> 16, top2 & 0xFFFFu);
#pragma unroll
            for (int sh = 1; sh < kLanes; sh <<= 1) {
              top = max(top, __shfl_xor_sync(0xffffffffu, top, sh));
            }
            // 2^14 over the power of two at or below the largest, at most 2^127.
            const int e = min(268 - static_cast<int>(top >> 7), 254);
            up = __uint_as_float(static_cast<uint32_t>(e) << 23);
          }
          float even = 0.f, odd = 0.f;
          uint8_t* dst = xs + m * p.x_pitch + (gr * (GROUP / 8) + t) * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t h[4] = {v[j].x, v[j].y, v[j].z, v[j].w};  // eight fp16, in order
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (kScaled) {
                h[k] = Elt<__half>::pack(__uint_as_float(h[k] << 16) * up,
                                         __uint_as_float(h[k] & 0xFFFF0000u) * up);
              }
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
              even += f.x;
              odd += f.y;
            }
            if (on) {
              *reinterpret_cast<uint4*>(dst + j * kLanes * 16) =
                  make_uint4(__byte_perm(h[0], h[2], 0x5410), __byte_perm(h[0], h[2], 0x7632),
                             __byte_perm(h[1], h[3], 0x5410), __byte_perm(h[1], h[3], 0x7632));
            }
          }
#pragma unroll
          for (int sh = 1; sh < kLanes; sh <<= 1) {
            even += __shfl_xor_sync(0xffffffffu, even, sh);
            odd += __shfl_xor_sync(0xffffffffu, odd, sh);
          }
          // (Finite ones cannot overflow: 128 fp16 numbers.)
          met |= !(fabsf(even + odd) <= 3.4e38f);
          if (on && t == 0) {
            float* at = sx + gr * kPlanes * (8 * NT) + m;
            // Offsets: 1024 for the pairs (0,4) and (2,6), 64 for the others.
            at[0] = ZP ? -(1024.f * even + 64.f * odd) : -(1032.f * even + 72.f * odd);
            if (ZP) at[8 * NT] = even + odd;
            if (kScaled) at[(kPlanes - 1) * 8 * NT] = 1.f / up;
          }
          m += step_m;
          gr += step_g;
          if (gr >= groups) {
            gr -= groups;
            ++m;
          }
        }
      }
      nonfinite |= __syncthreads_or(met);
      if (pv == v0 && ph == 0) w4_pdl_trigger();

      int off = w;  // this warp's next chunk, counted from the block's first
      for (int v = pv + halves * team; v < pe; v = next_block(v)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) total[mt][nt][e] = 0.f;
          }
        }
        for (; off < nch; off += T_) chunk(off);
        off -= nch;
        // The team's sum of the block, the warps in order.
        const float* sums = red + red_buf * kRedFloats;
        if (kRedBufs == 0) sums = reinterpret_cast<const float*>(smem + (s_dst - smem_u32(smem)));
        float4* mine = reinterpret_cast<float4*>(const_cast<float*>(sums) + (kRedBufs ? w * kFrag * 128 : 0));
        red_buf ^= 1;
        if (kRedBufs == 0 && lane == 0) s_free[warp] = s_dst - smem_u32(smem);
        __syncwarp();  // the slot's last chunk is read by all lanes
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mine[(mt * NT + nt) * 32 + lane] =
                make_float4(total[mt][nt][0], total[mt][nt][1], total[mt][nt][2], total[mt][nt][3]);
          }
        }
        team_sync();
        const bool up = p.silu && (v & 1);
        // A thread sums one lane's four values of a fragment; the warps that do
        // (fragments may be fewer than warps) change from block to block.
        for (int x = ((w + turn) & (T_ - 1)) * 32 + lane; x < kFrag * 32; x += 32 * T_) {
          float4* kept = reinterpret_cast<float4*>(acc) + (v - pv) * kFrag * 32 + x;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (ph > 0) y = *kept;
#pragma unroll 4
          for (int j = 0; j < T_; ++j) {
            const float4 z = kRedBufs ? reinterpret_cast<const float4*>(sums)[j * kFrag * 32 + x]
                                      : reinterpret_cast<const float4*>(smem + s_free[team * T_ + j])[x];
            y.x += z.x;
            y.y += z.y;
            y.z += z.z;
            y.w += z.w;
          }
          if (ph + 1 < p.phases) {
            *kept = y;
            continue;
          }
          // Fragment: (feature g, row 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1).
          const int f = x >> 5;
          const int feat = (p.silu ? v >> 1 : v) * kRows + (f / NT) * 16 + g;
          const int m = (f % NT) * 8 + 2 * c;
          if (nonfinite) y = w4_nonfinite4<T, GROUP>(p, feat, m, up, y);
          if (p.silu && !up) {
            reinterpret_cast<float4*>(gate)[x] = y;  // read back by this thread
          } else {
            if (up) {
              const float4 z = reinterpret_cast<const float4*>(gate)[x];
              y.x *= z.x / (1.f + expf(-z.x));
              y.y *= z.y / (1.f + expf(-z.y));
              y.z *= z.z / (1.f + expf(-z.z));
              y.w *= z.w / (1.f + expf(-z.w));
            }
            T* at = out + m * p.out_stride + feat;
            if (m < p.M && feat < p.N) at[0] = Elt<T>::from_f(y.x);
            if (m + 1 < p.M && feat < p.N) at[p.out_stride] = Elt<T>::from_f(y.y);
            if (m < p.M && feat + 8 < p.N) at[8] = Elt<T>::from_f(y.z);
            if (m + 1 < p.M && feat + 8 < p.N) at[p.out_stride + 8] = Elt<T>::from_f(y.w);
          }
        }
        if (!p.silu || up) ++turn;
        if (kRedBufs == 0) team_sync();  // the sums are taken before the slots are filled again
      }
    }
  }
}

// ── host side ────────────────────────────────────────────────────────────────

template <typename T, int GROUP, int NT, int MT, bool ZP>
int w4_launch(const W4Params& p, int grid, cudaStream_t s) {
  static std::once_flag flags[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(VMPS_ERR_CUDA, "device index %d", dev);
  std::call_once(flags[dev], [] {
    cudaFuncSetAttribute(w4_kernel<T, GROUP, NT, MT, ZP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         kW4SmemLimit);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, w4_kernel<T, GROUP, NT, MT, ZP>, p);
  if (e != cudaSuccess) {
    return fail(VMPS_ERR_CUDA, "w4_gemm: launch failed: %s", cudaGetErrorString(e));
  }
  return VMPS_OK;
}

template <typename T, int GROUP, bool ZP>
int w4_by_rows(const W4Params& p, int grid, cudaStream_t s) {
  switch (w4_nt(p.M)) {
    case 1: return w4_launch<T, GROUP, 1, 1, ZP>(p, grid, s);
    case 2: return w4_launch<T, GROUP, 2, 2, ZP>(p, grid, s);
    default: return w4_launch<T, GROUP, 4, 1, ZP>(p, grid, s);
  }
}

template <typename T, bool ZP>
int w4_by_group(int group, const W4Params& p, int grid, cudaStream_t s) {
  switch (group) {
    case 32: return w4_by_rows<T, 32, ZP>(p, grid, s);
    case 64: return w4_by_rows<T, 64, ZP>(p, grid, s);
    default: return w4_by_rows<T, 128, ZP>(p, grid, s);
  }
}

template <typename T>
int w4_by_zeros(int group, const W4Params& p, int grid, cudaStream_t s) {
  return p.zeros ? w4_by_group<T, true>(group, p, grid, s) : w4_by_group<T, false>(group, p, grid, s);
}

}  // namespace
}  // namespace vmps

using namespace vmps;

extern "C" int vmps_w4_gemm_supported(int M, int N, int K, int group_size) {
  if (M < 0 || M > kW4MaxRows || N <= 0 || K <= 0) return 0;
  if (group_size != 32 && group_size != 64 && group_size != 128) return 0;
  if (K % group_size || K > kW4MaxK) return 0;
  // Indices into the scales (of up to 2 N rows) are 31 bits.
  return 2 * static_cast<int64_t>(N) * (K / group_size) <= 0x7fffffff ? 1 : 0;
}

extern "C" int vmps_w4_gemm(void* out, int64_t out_row_stride, const void* x, int64_t x_row_stride,
                            const void* codes, const void* scales, const void* zeros, int M, int N,
                            int K, int group_size, int silu_mul, int dtype, void* stream) {
  const char* what = "w4_gemm";
  clear_error();
  if (dtype != VMPS_DTYPE_F16 && dtype != VMPS_DTYPE_BF16) {
    return fail(VMPS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  }
  if (!vmps_w4_gemm_supported(M, N, K, group_size)) {
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
  const int rows = 16 * w4_mt(M);
  W4Params p;
  p.out = out;
  p.out_stride = out_row_stride;
  p.x = x;
  p.x_stride = x_row_stride;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.M = M;
  p.N = N;
  p.K = K;
  p.ng = K / group_size;
  p.silu = silu_mul ? 1 : 0;
  p.blocks = (N + rows - 1) / rows;
  const int grid = p.blocks < sms ? p.blocks : sms;
  if (!w4_plan(&p, M, K, group_size, p.silu != 0, w4_planes(dtype != VMPS_DTYPE_F16, zeros != nullptr),
               (p.blocks + grid - 1) / grid * (p.silu ? 2 : 1))) {
    return fail(VMPS_ERR_UNSUPPORTED, "%s: no shared-memory plan for M=%d K=%d", what, M, K);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == VMPS_DTYPE_F16 ? w4_by_zeros<__half>(group_size, p, grid, s)
                                 : w4_by_zeros<__nv_bfloat16>(group_size, p, grid, s);
}
