// The work split of the tree attention: arithmetic on the lengths that every CTA
// does for itself, plain C++ so that it can be checked without a GPU.
#pragma once

#include <stdint.h>

#include "vmps_hd.h"

namespace vmps {

constexpr int kTtKeys = 64;  // keys per tile
// A sequence's start costs a share about four tiles: with 2 in place of 4, 32
// ragged sequences took 80.5 us for 77.9 and one of 8000 slots 21.5 for 19.8;
// with 6, 77.3 and 20.3 (8 kv heads, head size 128).
constexpr int kTileWeight = 4;
constexpr int kSegWeight = 4 * kTileWeight;
// Weight of a share, at least.  Short calls gain from small pieces until the
// join costs as much: one sequence of 1000 slots takes 17.4 us with 8 tiles,
// 13.7 with 3, 13.3 with 2; four of them (8 kv heads) 21.0, 17.4 and 17.6.
constexpr int kMinShare = 3 * kTileWeight;
// Contexts up to this many tiles are not cut, which saves the second launch:
// one sequence of 500 slots takes 13.1 us whole and 14.0 cut, 32 of them 17.7
// and 32.4; of 1000 slots one takes 19.1 whole and 13.7 cut.
constexpr int kWholeTiles = 8;

// A sequence with query rows has at least one tile (its rows are written even
// if it holds no slot).
VMPS_HD int tree_tiles(int n) { return n > 0 ? (n + kTtKeys - 1) / kTtKeys : 1; }

// Weight in row tile index rt of a sequence packed as tiles << 8 | row tiles.
VMPS_HD int tree_weight(int packed, int rt) {
  return (packed & 255) > rt ? (packed >> 8) * kTileWeight + kSegWeight : 0;
}

// Quotient of non-negative numbers: 32-bit where both fit (four times faster).
VMPS_HD long long tree_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Largest s in [0, n) with pref[s] <= f (pref non-decreasing, pref[0] = 0).
VMPS_HD int tree_find(const int* pref, int n, int f) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pref[mid] <= f) lo = mid; else hi = mid;
  }
  return lo;
}

// Weight of a share of `total` (of all row tile indices with work, `used` of
// them).  Row tile indices start on a CTA of their own, which can leave up to
// used - 1 shares partly empty.  Contexts that are not cut start a CTA each
// while there are CTAs left.
VMPS_HD long long tree_chunk(long long total, int used, int n_cta, int whole) {
  const int div = n_cta - (used > 0 ? used - 1 : 0);
  const long long chunk = tree_div(total + div - 1, div);
  const long long least = whole ? 1 : kMinShare;
  return chunk < least ? least : chunk;
}

struct TreePos {  // a tile of a row tile's linear order
  int kvh, s, j;
};

// What a CTA does: row tile index, its place among that index's CTAs, its share.
struct TreeShare {
  int rt;
  int first_cta;      // first CTA of this row tile index
  long long chunk;    // weight of a share: of all row tile indices and kv heads, so above 31 bits
                      // for tables of hundreds of millions of slots
  TreePos begin, end; // tiles [begin, end)
};

// The share of tiles before weighted position w.
VMPS_HD TreePos tree_pos(const int* wpref, int num_seqs, int n_kv, int whole, long long w) {
  TreePos r;
  const int wt = wpref[num_seqs];
  if (w >= static_cast<long long>(n_kv) * wt) {
    r.kvh = n_kv;
    r.s = 0;
    r.j = 0;
    return r;
  }
  r.kvh = static_cast<int>(tree_div(w, wt));
  const int f = static_cast<int>(w - static_cast<long long>(r.kvh) * wt);
  r.s = tree_find(wpref, num_seqs, f);
  const int off = f - wpref[r.s];
  const int tiles = (wpref[r.s + 1] - wpref[r.s] - kSegWeight) / kTileWeight;
  r.j = off <= kSegWeight ? 0 : (off - kSegWeight + kTileWeight - 1) / kTileWeight;
  if (whole && off > 0) r.j = tiles;
  return r;
}

// Walks the segments (runs of tiles of one sequence and kv head) of a share.
struct TreeWalk {
  TreePos at;
  int j1;  // tiles [at.j, j1) of the segment
  int tiles;
  bool valid;

  VMPS_HD void settle(const int* wpref, int num_seqs, const TreePos& end) {
    for (;;) {
      if (at.kvh > end.kvh || (at.kvh == end.kvh && at.s > end.s)) break;
      const bool last = at.kvh == end.kvh && at.s == end.s;
      if (last && end.j <= at.j) break;
      const int w = wpref[at.s + 1] - wpref[at.s];
      if (w > 0) {
        tiles = (w - kSegWeight) / kTileWeight;
        j1 = last && end.j < tiles ? end.j : tiles;
        if (j1 > at.j) {
          valid = true;
          return;
        }
      }
      if (++at.s == num_seqs) {
        at.s = 0;
        ++at.kvh;
      }
      at.j = 0;
    }
    valid = false;
  }
  VMPS_HD void start(const int* wpref, int num_seqs, const TreeShare& sh) {
    at = sh.begin;
    settle(wpref, num_seqs, sh.end);
  }
  VMPS_HD void next(const int* wpref, int num_seqs, const TreeShare& sh) {
    if (++at.s == num_seqs) {
      at.s = 0;
      ++at.kvh;
    }
    at.j = 0;
    settle(wpref, num_seqs, sh.end);
  }
};

// The CTA (within its row tile index) that owns tile j of the segment.
VMPS_HD int tree_owner(const int* wpref, int num_seqs, const TreeShare& sh, int kvh, int s, int j) {
  const long long w = static_cast<long long>(kvh) * wpref[num_seqs] + wpref[s] + kSegWeight +
                      static_cast<long long>(j) * kTileWeight;
  return static_cast<int>(tree_div(w, sh.chunk));
}

}  // namespace vmps
