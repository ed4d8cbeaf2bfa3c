// How a product with 4-bit weights divides a CTA's shared memory and its work:
// plain arithmetic that any C++ compiler takes, so that it can be checked without
// a GPU.
#pragma once

#include "vmps_hd.h"

namespace vmps {

constexpr int kW4MaxRows = 32;
constexpr int kW4Warps = 16;
constexpr int kW4Threads = 32 * kW4Warps;
constexpr int kW4Depth = 2;  // ring slots per warp: one chunk in flight, one in use
constexpr int kW4SmemLimit = 226 * 1024;  // dynamic; up to 1024 static bytes come on top
// Chunk numbers times codes per chunk stay in 31 bits.
constexpr int kW4MaxK = 0x7fffffff - 1023;

// Activation tiles of 8 rows and 16-feature tiles that share them.
VMPS_HD constexpr int w4_nt(int M) { return M <= 8 ? 1 : (M <= 16 ? 2 : 4); }
VMPS_HD constexpr int w4_mt(int M) { return M > 8 && M <= 16 ? 2 : 1; }

// Codes of a chunk (kRows rows x 2 * bytes / kRows codes): the larger amortises
// more, but with more than one activation tile the activations need the room.
VMPS_HD constexpr int w4_chunk_bytes(int nt) { return nt == 1 ? 4096 : 2048; }
VMPS_HD constexpr int w4_chunk_codes(int M) { return w4_chunk_bytes(w4_nt(M)) * 2 / (16 * w4_mt(M)); }

// Buffers of partial sums beside the rings: with two a team meets once per
// block.  With more than one activation tile there is no room for them; a
// warp's sums then go to its free ring slot, and the team meets twice.
VMPS_HD constexpr int w4_red_bufs(int nt) { return nt == 1 ? 2 : 0; }

// Per group and activation row: what its sum starts from, [sum x,] [what its
// sum is multiplied by].
VMPS_HD constexpr int w4_planes(bool scaled, bool zp) { return 1 + (zp ? 1 : 0) + (scaled ? 1 : 0); }

struct W4Plan {
  int chunks;            // of K (the last may be partial)
  int slice;             // chunks per phase
  int phases;
  int panel;             // blocks a CTA carries through the phases at once
  int team;              // warps that share a block (a power of two)
  int x_pitch;           // bytes between activation rows in shared memory
  int x_bytes, sx_bytes;
  int smem;              // dynamic shared memory of a CTA, bytes
};

// The plan with the fewest bytes of X staged per CTA (phases times panels) that
// leaves room for everything else; false if there is none.  `cta_blocks`: blocks
// of 16 w4_mt(M) features of the busiest CTA, gate and up halves counted apart.
// Sizes are 64-bit until they are known to fit: M rows of a long K pass 31 bits.
inline bool w4_plan(W4Plan* p, int M, int K, int group, bool silu, int planes, int cta_blocks) {
  const int nt = w4_nt(M), mt = w4_mt(M), codes = w4_chunk_codes(M);
  const int halves = silu ? 2 : 1;
  p->chunks = (K + codes - 1) / codes;
  // A warp should take about 16 KB of a block (its share of the block's fixed
  // costs: with teams of 4 instead of 8 the LM head at 16 rows took 80 us for
  // 88), but all warps should have a block.
  const int few = 16384 / w4_chunk_bytes(nt);
  p->team = 1;
  while (p->team < kW4Warps && (p->team * few < p->chunks || p->team * (cta_blocks / halves) < kW4Warps)) {
    p->team *= 2;
  }
  const int block = mt * nt * 512;  // bytes of a block's sums
  const int fixed = kW4Warps * kW4Depth * w4_chunk_bytes(nt) +
                    (w4_red_bufs(nt) * kW4Warps + (silu ? kW4Warps / p->team : 0)) * block;
  long long best = -1;
  // No slice above this many chunks fits, so fewer phases need not be looked at.
  const int most = (kW4SmemLimit - fixed) / (M * codes * 2) + 1;
  for (int phases = (p->chunks + most - 1) / most; phases <= p->chunks; ++phases) {
    const int slice = (p->chunks + phases - 1) / phases;
    if ((p->chunks + slice - 1) / slice != phases) continue;
    const long long pitch = static_cast<long long>(slice) * codes * 2 + 64;  // 64 mod 128: rows g and g + 1 fill all banks
    const long long x_bytes = (M * pitch + 127) / 128 * 128;
    const long long sx_bytes = static_cast<long long>(slice) * (codes / group) * 8 * nt * 4 * planes;
    const long long left = kW4SmemLimit - fixed - x_bytes - sx_bytes;
    int panel = cta_blocks;
    if (left < 0) continue;
    if (phases > 1) {
      panel = static_cast<int>(left) / block / halves * halves;
      if (panel < halves) continue;
      if (panel > cta_blocks) panel = cta_blocks;
    }
    const long long cost = phases == 1 ? 0 : ((static_cast<long long>(cta_blocks) + panel - 1) / panel) *
                                                 (p->chunks + 8LL * phases);
    if (best < 0 || cost < best) {
      best = cost;
      p->slice = slice;
      p->phases = phases;
      p->panel = panel;
      p->x_pitch = static_cast<int>(pitch);
      p->x_bytes = static_cast<int>(x_bytes);
      p->sx_bytes = static_cast<int>(sx_bytes);
      p->smem = fixed + p->x_bytes + p->sx_bytes + (phases > 1 ? panel * block : 0);
    }
    if (panel == cta_blocks) break;  // more phases only cost more
  }
  return best >= 0;
}

}  // namespace vmps
