// The work split of decode attention over the 8-bit cache: arithmetic on the
// lengths that every CTA does for itself, plain C++ so that it can be checked
// without a GPU.
//
// The tiles of all sequences and head groups are laid end to end (head group,
// sequence, tile), a sequence's start weighing as much as some tiles, and cut
// into equal contiguous shares, one per CTA.  A sequence cut between CTAs has a
// piece in each CTA of a run; a CTA has at most two pieces of cut sequences, the
// end of one (slot 0) and the start of another (slot 1).
#pragma once

#include <stdint.h>

#include "vmps_hd.h"

namespace vmps {

constexpr int kC8TileWeight = 4;
// A sequence's start costs a share about two tiles: with 1 in place of 2, 64
// ragged sequences took 20.0 us for 19.4 and 16 x 1..8192 43.6 for 42.2; with
// 3, 256 x 511..1537 99.3 for 96.8.
constexpr int kC8SegWeight = 2 * kC8TileWeight;
// Weight of a share, at least: with twice as much, one sequence of 128 tokens
// took 9.8 us for 6.5 and one of 1024 12.1 for 10.2 (8 kv heads).
constexpr int kC8MinShare = 2 * kC8TileWeight;

struct C8Shape {
  int num_seqs;
  int groups;       // head groups
  int n_cta;
  long long chunk;  // weight of a share
};

VMPS_HD long long c8_div(long long a, long long b) {
  // 32-bit where both fit: four times faster on the GPU.
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Tiles of 2^shift tokens.
VMPS_HD int c8_tiles(int len, int shift) { return len > 0 ? ((len - 1) >> shift) + 1 : 0; }

VMPS_HD int c8_weight(int tiles) { return tiles > 0 ? tiles * kC8TileWeight + kC8SegWeight : 0; }

// Weight of a share: of `total`, the weight of one head group's sequences.
VMPS_HD long long c8_chunk(long long total, int groups, int n_cta) {
  const long long chunk = c8_div(total * groups + n_cta - 1, n_cta);
  return chunk < kC8MinShare ? kC8MinShare : chunk;
}

struct C8Pos {  // a tile in the linear order
  int hg, s, j;
};

// Weighted position w as a head group and a position in its sequences (hg is the
// number of groups behind the last).
struct C8Cut {
  int hg, at;
};

VMPS_HD C8Cut c8_cut(int total, int groups, long long w) {
  C8Cut r;
  r.hg = groups;
  r.at = 0;
  if (w >= static_cast<long long>(groups) * total) return r;
  r.hg = groups == 1 ? 0 : static_cast<int>(c8_div(w, total));
  r.at = static_cast<int>(w - static_cast<long long>(r.hg) * total);
  return r;
}

// The first tile at or after weighted position `off` of a sequence.
VMPS_HD int c8_tile_at(int off) {
  return off <= kC8SegWeight ? 0 : (off - kC8SegWeight + kC8TileWeight - 1) / kC8TileWeight;
}

// The CTA that has tile j of the sequence.
VMPS_HD int c8_owner(const int* wpref, const C8Shape& sh, int hg, int s, int j) {
  const long long w = static_cast<long long>(hg) * wpref[sh.num_seqs] + wpref[s] + kC8SegWeight +
                      static_cast<long long>(j) * kC8TileWeight;
  return static_cast<int>(c8_div(w, sh.chunk));
}

// Walks the segments (runs of tiles of one sequence and head group) of a share.
struct C8Walk {
  int hg, s, j0, j1;  // tiles [j0, j1) of the segment
  int tiles;          // of the whole sequence
  bool valid;

  VMPS_HD void settle(const int* wpref, const C8Shape& sh, const C8Pos& end) {
    valid = false;
    while (hg < end.hg || (hg == end.hg && s <= end.s)) {
      const bool last = hg == end.hg && s == end.s;
      if (last && end.j <= j0) return;
      const int w = wpref[s + 1] - wpref[s];
      if (w > 0) {
        tiles = (w - kC8SegWeight) / kC8TileWeight;
        j1 = last && end.j < tiles ? end.j : tiles;
        if (j1 > j0) {
          valid = true;
          return;
        }
      }
      step(sh);
    }
  }
  VMPS_HD void step(const C8Shape& sh) {
    if (++s == sh.num_seqs) {
      s = 0;
      ++hg;
    }
    j0 = 0;
  }
  VMPS_HD void start(const int* wpref, const C8Shape& sh, const C8Pos& begin, const C8Pos& end) {
    hg = begin.hg;
    s = begin.s;
    j0 = begin.j;
    settle(wpref, sh, end);
  }
  VMPS_HD void next(const int* wpref, const C8Shape& sh, const C8Pos& end) {
    step(sh);
    settle(wpref, sh, end);
  }
};

// Pieces are joined by the CTA that finishes last.  Runs of many pieces are
// joined in two rounds, groups of 16 first, so that no one CTA reads them all.
constexpr int kC8OneRound = 24;

VMPS_HD int c8_join_group(int pieces) { return pieces <= kC8OneRound ? pieces : 16; }

}  // namespace vmps
