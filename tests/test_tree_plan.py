"""The work split of the tree attention (``csrc/tree_plan.h``), compiled as plain C++.

Every CTA's share is worked out as the kernel does it.  Together the shares
hold every tile of every sequence, kv head and row tile once; the CTA that
``tree_owner`` names for a piece's ends is the one that has it; a CTA has at
most two pieces of cut sequences, one in each of its two slots; and the CTA
after the one where a cut sequence begins has its second piece.
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
#include <vector>
#include "tree_plan.h"
using namespace vmps;
// packed: tiles << 8 | row tiles of every sequence.  0, or which property failed.
extern "C" int check(int num_seqs, const int* packed, int n_kv, int row_tiles, int n_cta, int whole,
                     long long* chunk_out) {
  std::vector<long long> weight(row_tiles);
  long long total = 0;
  int used = 0;
  for (int rt = 0; rt < row_tiles; ++rt) {
    for (int s = 0; s < num_seqs; ++s) weight[rt] += tree_weight(packed[s], rt);
    if (weight[rt] > 0x7fffffffLL) return 1;  // the host refuses such calls
    if (weight[rt] > 0) { ++used; total += weight[rt] * n_kv; }
  }
  const long long chunk = tree_chunk(total, used, n_cta, whole);
  *chunk_out = chunk;
  std::vector<int> wpref(num_seqs + 1);
  std::vector<int> done((size_t)row_tiles * n_kv * num_seqs, 0);  // tiles covered so far
  std::vector<int> first_piece(done.size(), -1);
  int first = 0;
  for (int rt = 0; rt < used; ++rt) {
    const int n = (int)tree_div(weight[rt] * n_kv + chunk - 1, chunk);
    if (first + n > n_cta) return 2;
    for (int s = 0; s < num_seqs; ++s) wpref[s + 1] = wpref[s] + tree_weight(packed[s], rt);
    for (int b = first; b < first + n; ++b) {
      TreeShare sh;
      sh.rt = rt;
      sh.first_cta = first;
      sh.chunk = chunk;
      sh.begin = tree_pos(wpref.data(), num_seqs, n_kv, whole, (b - first) * chunk);
      sh.end = tree_pos(wpref.data(), num_seqs, n_kv, whole, (b - first + 1) * chunk);
      int slots = 0;
      TreeWalk w;
      w.start(wpref.data(), num_seqs, sh);
      for (; w.valid; w.next(wpref.data(), num_seqs, sh)) {
        const int s = w.at.s, kvh = w.at.kvh, j0 = w.at.j, j1 = w.j1;
        if (w.tiles != packed[s] >> 8) return 3;
        int& at = done[((size_t)rt * n_kv + kvh) * num_seqs + s];
        if (at != j0 || j1 <= j0) return 4;
        at = j1;
        if (j0 == 0 && j1 == w.tiles) continue;
        if (whole) return 5;
        if (tree_owner(wpref.data(), num_seqs, sh, kvh, s, j0) + first != b) return 6;
        if (tree_owner(wpref.data(), num_seqs, sh, kvh, s, j1 - 1) + first != b) return 7;
        const int c0 = tree_owner(wpref.data(), num_seqs, sh, kvh, s, 0) + first;
        int& before = first_piece[((size_t)rt * n_kv + kvh) * num_seqs + s];
        if (j0 == 0) {
          if (c0 != b) return 8;
          before = b;
        } else {
          if (before < 0 || c0 + 1 > b) return 9;
          if (before + 1 != b) return 10;  // a piece in every CTA up to the last
          before = b;
        }
        const int slot = c0 == b ? 1 : 0;
        if (slots & (1 << slot)) return 11;
        slots |= 1 << slot;
      }
    }
    for (int kvh = 0; kvh < n_kv; ++kvh) {
      for (int s = 0; s < num_seqs; ++s) {
        const int want = (packed[s] & 255) > rt ? packed[s] >> 8 : 0;
        if (done[((size_t)rt * n_kv + kvh) * num_seqs + s] != want) return 12;
      }
    }
    first += n;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "no C++ compiler"
    d = tmp_path_factory.mktemp("tree_plan")
    (d / "plan.cpp").write_text(HARNESS)
    lib = str(d / "plan.so")
    subprocess.run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-I", CSRC, "-o", lib,
                    str(d / "plan.cpp")], check=True)
    fn = ctypes.CDLL(lib).check

    def call(seqs, n_kv, n_cta=296, whole=False):
        """``seqs``: (tiles, row tiles) each; returns (failed property or 0, chunk)."""
        packed = (ctypes.c_int * len(seqs))(*[(t << 8) | r for t, r in seqs])
        chunk = ctypes.c_longlong()
        rc = fn(len(seqs), packed, n_kv, max(1, max(r for _, r in seqs)), n_cta, int(whole),
                ctypes.byref(chunk))
        return rc, chunk.value
    return call


def test_shares_hold_every_tile_once(check):
    rng = random.Random(1)
    for _ in range(1500):
        n = rng.choice([1, 1, 2, 3, 8, 40, 300])
        top = rng.choice([1, 3, 8, 60, 2000, 40000])
        rows = rng.choice([1, 1, 2, 5, 128])
        seqs = [(rng.randint(1, top), rng.randint(0, rows)) for _ in range(n)]
        whole = top <= 8 and rng.random() < 0.7
        rc, _ = check(seqs, rng.choice([1, 2, 4, 8, 64]), rng.choice([296, 264, 300]), whole)
        assert rc == 0, (rc, seqs[:5])


def test_shares_above_31_bits(check):
    """Tables of 2^24 blocks, as many row tiles and kv heads as there can be."""
    rc, chunk = check([(2 ** 22, 128)] * 4, 64)
    assert chunk > 2 ** 31
    assert rc == 0
    rc, chunk = check([(2 ** 22 - 5, 128), (2 ** 22, 100), (77, 128), (2 ** 21, 3)] * 20, 64)
    assert chunk > 2 ** 31
    assert rc == 0
