"""The work split of decode attention over the 8-bit cache (``csrc/cache8_plan.h``),
compiled as plain C++.

Every CTA's share is worked out as the kernel does it.  Together the shares hold
every tile of every sequence and head group once; the CTAs that ``c8_owner``
names for a cut sequence's ends are those that have them, with a piece in every
CTA between; a CTA has at most one piece in each of its two slots; and the
groups in which a run of pieces is joined have at most 32 members and are at
most 32, for up to 512 pieces.
"""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "vllm_mps_b200", "csrc")
HARNESS = """
#include <algorithm>
#include <vector>
#include "cache8_plan.h"
using namespace vmps;
// The kernel's threads look at their sequences, one finds the cut in its own.
static C8Pos pos(const std::vector<int>& wpref, const C8Shape& sh, long long w) {
  const C8Cut cut = c8_cut(wpref[sh.num_seqs], sh.groups, w);
  C8Pos r = {cut.hg, 0, 0};
  if (cut.hg == sh.groups) return r;
  const int s = (int)(std::upper_bound(wpref.begin(), wpref.end(), cut.at) - wpref.begin()) - 1;
  r.s = s;
  r.j = c8_tile_at(cut.at - wpref[s]);
  return r;
}
extern "C" int check(int num_seqs, const int* lens, int shift, int groups, int n_cta) {
  std::vector<int> wpref(num_seqs + 1, 0);
  long long total = 0;
  for (int s = 0; s < num_seqs; ++s) {
    total += c8_weight(c8_tiles(lens[s], shift));
    if (total > 0x7fffffffLL) return 1;  // the host refuses such calls
    wpref[s + 1] = (int)total;
  }
  C8Shape sh;
  sh.num_seqs = num_seqs;
  sh.groups = groups;
  sh.n_cta = n_cta;
  sh.chunk = c8_chunk(total, groups, n_cta);
  std::vector<int> done((size_t)groups * num_seqs, 0), piece(done.size(), -1);
  for (int b = 0; b < n_cta; ++b) {
    const C8Pos begin = pos(wpref, sh, b * sh.chunk), end = pos(wpref, sh, (b + 1) * sh.chunk);
    int slots = 0;
    C8Walk w;
    for (w.start(wpref.data(), sh, begin, end); w.valid; w.next(wpref.data(), sh, end)) {
      const size_t at = (size_t)w.hg * num_seqs + w.s;
      if (w.tiles != c8_tiles(lens[w.s], shift)) return 2;
      if (done[at] != w.j0 || w.j1 <= w.j0) return 3;
      done[at] = w.j1;
      if (w.j0 == 0 && w.j1 == w.tiles) continue;
      const int c0 = c8_owner(wpref.data(), sh, w.hg, w.s, 0);
      const int c1 = c8_owner(wpref.data(), sh, w.hg, w.s, w.tiles - 1);
      if (c0 >= c1 || c1 >= n_cta) return 4;
      if (w.j0 == 0 ? b != c0 : piece[at] + 1 != b) return 5;
      if ((w.j1 == w.tiles) != (b == c1)) return 6;
      piece[at] = b;
      const int slot = b == c0;
      if (slots & (1 << slot)) return 7;
      slots |= 1 << slot;
    }
  }
  for (int g = 0; g < groups; ++g)
    for (int s = 0; s < num_seqs; ++s)
      if (done[(size_t)g * num_seqs + s] != c8_tiles(lens[s], shift)) return 8;
  return 0;
}
extern "C" int join_group(int pieces) { return c8_join_group(pieces); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "no C++ compiler"
    d = tmp_path_factory.mktemp("cache8_plan")
    (d / "plan.cpp").write_text(HARNESS)
    out = str(d / "plan.so")
    subprocess.run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-I", CSRC, "-o", out,
                    str(d / "plan.cpp")], check=True)
    return ctypes.CDLL(out)


def _check(lib, lens, tile=16, groups=1, n_cta=296):
    return lib.check(len(lens), (ctypes.c_int * len(lens))(*lens), tile.bit_length() - 1, groups, n_cta)


def test_shares_hold_every_tile_once(lib):
    rng = random.Random(1)
    for _ in range(2000):
        n = rng.choice([1, 1, 2, 3, 8, 64, 300, 4096])
        top = rng.choice([1, 16, 40, 300, 5000, 200000])
        lens = [rng.randint(0, top) for _ in range(n)]
        rc = _check(lib, lens, rng.choice([16, 32, 64, 128]), rng.choice([1, 1, 2, 11, 64]),
                    rng.choice([296, 148, 264]))
        assert rc == 0, (rc, lens[:5])


def test_longest_tables(lib):
    assert _check(lib, [2 ** 31 - 1] * 3, 16, 64) == 0
    assert _check(lib, [0, 2 ** 31 - 1, 0, 1], 16, 64) == 0
    assert _check(lib, [0, 0]) == 0


def test_groups_of_pieces_that_are_joined(lib):
    for pieces in range(2, 513):
        g = lib.join_group(pieces)
        assert 1 < g <= pieces and g <= 32 and -(-pieces // g) <= 32
        assert g == pieces or pieces > 24
