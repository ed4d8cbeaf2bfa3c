"""The shared-memory plan of the 4-bit products (``csrc/w4_plan.h``), compiled as plain C++."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "vllm_mps_b200", "csrc")
HARNESS = """
#include "w4_plan.h"
extern "C" int plan(int M, int K, int group, int silu, int planes, int cta_blocks, int* out) {
  vmps::W4Plan p;
  if (!vmps::w4_plan(&p, M, K, group, silu != 0, planes, cta_blocks)) return 0;
  const int v[9] = {p.chunks, p.slice, p.phases, p.panel, p.team, p.x_pitch, p.x_bytes, p.sx_bytes, p.smem};
  for (int i = 0; i < 9; ++i) out[i] = v[i];
  return 1;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "no C++ compiler"
    d = tmp_path_factory.mktemp("w4_plan")
    (d / "plan.cpp").write_text(HARNESS)
    lib = str(d / "plan.so")
    subprocess.run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-I", CSRC, "-o", lib,
                    str(d / "plan.cpp")], check=True)
    fn = ctypes.CDLL(lib).plan

    def call(*args):
        out = (ctypes.c_int * 9)()
        if not fn(*args, out):
            return None
        return dict(zip(("chunks", "slice", "phases", "panel", "team", "x_pitch", "x_bytes",
                         "sx_bytes", "smem"), out))
    return call


MAX_K = 2 ** 31 - 1024  # what vmps_w4_gemm_supported accepts


@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("silu", [0, 1])
@pytest.mark.parametrize("K", [32, 2048, 14336, 16384, 131072, 2 ** 22, 2 ** 25, 2 ** 26, 2 ** 26 + 256,
                               2 ** 27, 3 * 2 ** 26, 2 ** 30, MAX_K // 128 * 128])
def test_what_is_staged_fits(plan, M, silu, K):
    """Every byte that the kernel writes, counted in whole numbers, is inside what it asks for."""
    nt = 1 if M <= 8 else 2 if M <= 16 else 4
    mt = 2 if nt == 2 else 1
    chunk = 4096 if nt == 1 else 2048
    codes = chunk * 2 // (16 * mt)
    for group in (32, 64, 128):
        if K % group:
            continue
        for planes in (1, 2, 3):
            for cta_blocks in (1 + silu, 6 * (1 + silu), 866):
                p = plan(M, K, group, silu, planes, cta_blocks)
                assert p is not None
                assert p["chunks"] == -(-K // codes)
                assert 1 <= p["slice"] <= p["chunks"]
                assert p["phases"] == -(-p["chunks"] // p["slice"])
                assert p["team"] in (1, 2, 4, 8, 16)
                assert 1 + silu <= p["panel"] <= cta_blocks and p["panel"] % (1 + silu) == 0
                # A row of a slice and 64 bytes that keep rows off each other's banks.
                assert p["x_pitch"] == 2 * codes * p["slice"] + 64
                assert M * p["x_pitch"] <= p["x_bytes"] <= M * p["x_pitch"] + 127
                assert p["sx_bytes"] == p["slice"] * (codes // group) * 8 * nt * 4 * planes
                block = mt * nt * 512
                used = 16 * 2 * chunk + p["x_bytes"] + p["sx_bytes"]
                used += (2 * 16 if nt == 1 else 0) * block     # partial sums
                used += (16 // p["team"] if silu else 0) * block
                used += (p["panel"] if p["phases"] > 1 else 0) * block
                assert p["smem"] == used <= 226 * 1024


def test_supported_lengths():
    from vllm_mps_b200 import kernels as K

    assert K.w4_gemm_supported(32, 1, MAX_K // 128 * 128, 128)
    assert not K.w4_gemm_supported(1, 1, MAX_K + 1024 - 128, 128)  # chunk ends would pass 31 bits
