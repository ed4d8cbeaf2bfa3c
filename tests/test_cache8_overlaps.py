"""Outputs in their inputs' place are refused (CPU: host arithmetic and C entries)."""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest

from test_cache8_host import A, _c_store, _lib
from vllm_mps_b200 import kernels as K

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "vllm_mps_b200", "csrc")
HARNESS = """
#include "rows_overlap.h"
extern "C" int overlap(long a, long as, long ar, long b, long bs, long br, long rows) {
  return vmps::rows_overlap((void*)a, as, ar, (void*)b, bs, br, rows);
}
"""


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "o.cpp").write_text(HARNESS)
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o",
                    str(d / "o.so"), str(d / "o.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "o.so")).overlap
    fn.argtypes = [ctypes.c_long] * 7
    return fn


def _bytes(start, stride, row, rows):
    return {start + i * stride + j for i in range(rows) for j in range(row)}


def test_every_overlap_is_seen(overlap):
    """Against sets of bytes; rows of one stride, and contiguous ones, are told apart exactly."""
    rng = random.Random(1)
    seen = [0, 0, 0]
    for _ in range(40000):
        rows = rng.choice([0, 1, 1, 2, 3, 5])
        ar, br = rng.choice([0, 1, 2, 3, 6]), rng.choice([1, 2, 3, 6])
        as_, bs = ar + rng.choice([0, 0, 1, 4, 12]), br + rng.choice([0, 0, 1, 4, 12])
        if rng.random() < 0.5:
            bs = as_ = max(as_, bs)
        a, b = 1000, 1000 + rng.randint(-40, 40)
        want = bool(_bytes(a, as_, ar, rows) & _bytes(b, bs, br, rows))
        got = bool(overlap(a, as_, ar, b, bs, br, rows))
        assert got or not want
        seen[0] += want
        seen[1] += not got
        if as_ == bs or rows == 1:
            assert got == want, (rows, a, as_, ar, b, bs, br)
            seen[2] += 1
    assert min(seen) > 5000


@pytest.mark.parametrize("change", [
    # rows of 512 bytes of q and q_out, 256 of k and v, three of them
    dict(q_out=A + 16, q=A, k=1 << 24, v=1 << 25),           # between q's elements
    dict(q_out=A, q=A, qs=512, qos=256, k=1 << 24, v=1 << 25),  # q's first row, then its gap
    dict(q_out=A, q=1 << 24, k=A + 1024, v=1 << 25),         # k from q_out's third row on
    dict(q_out=A + 512, q=A, qos=640, qs=640, k=A + 512, ks=640, v=A + 1024, vs=640),  # in k's place
    dict(q_out=A + 512 + 2 * 1280, q=A, qs=640, qos=640, k=1 << 24, v=A + 512, vs=640),
])
def test_store_refuses_overlaps(change):
    assert _c_store(**{**change, "eps": 1e-6}) == -1
    assert b"overlaps" in _lib().vmps_last_error()


@pytest.mark.parametrize("out", [A, A + 16, A + 1536 - 16, A - 1536 + 16])
def test_decode_refuses_overlaps(out):
    a = dict(out=out, q=A, qs=256, codes=A, scales=A, bt=A, mb=4, lens=A, B=3, n_q=4, n_kv=2, d=64,
             bs=16, nb=2, scale=0.125, ws=A, wsb=1 << 40, fmt=K.VMPS_CACHE_INT8, dtype=0, stream=None)
    assert _lib().vmps_paged_decode_attention_cache8(*a.values()) == -1
    assert b"overlaps" in _lib().vmps_last_error()
