"""The 8-bit pool's host-side access and its swap space (CPU: torch indexing alone)."""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200.kernels import KVCache8
from vllm_mps_b200.memory.cuda_memory_pool import CUDACache8Pool, CUDAMemoryPool, SwapSpace

FORMATS = [torch.int8, torch.float8_e4m3fn]
# A value is within half a code step of what is read: 1/254 of its row's largest (int8),
# 2^-4 of itself (e4m3); and the 16-bit rounding of what is returned (fp16 2^-11).
STEP = {torch.int8: 1 / 254 + 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4 + 2.0 ** -10}


def _pool(fmt, layers=None, blocks=6):
    return CUDACache8Pool(blocks, 16, 2, 64, torch.float16, "cpu", layers, fmt)


def _near(got, want, fmt):
    top = want.abs().amax(-1, keepdim=True)
    return ((got.float() - want.float()).abs() <= STEP[fmt] * top).all()


@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("fmt", FORMATS)
def test_write_read_gather_copy(fmt, layers):
    pool = _pool(fmt, layers)
    layer = 0 if layers is None else 2
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((2, 20, 2, 64), generator=g).half()
    table = [4, 1]
    for t in range(20):
        pool.write_kv(table[t // 16], t % 16, k[t], v[t], layer)
    got = pool.read_kv(1, 3, layer)
    assert got[0].dtype == torch.float16 and _near(got[0], k[19], fmt) and _near(got[1], v[19], fmt)
    kk, vv = pool.gather_blocks(table, layer)
    assert kk.shape == (32, 2, 64) and _near(kk[:20], k, fmt) and _near(vv[:20], v, fmt)
    assert (kk[20:] == 0).all()
    bk, bv = pool.gather_blocks_batched([[4], table, []], [5, 20, 0], 24, layer)
    assert bk.shape == (3, 24, 2, 64) and torch.equal(bk[1, :20], kk[:20]) and (bk[2] == 0).all()
    assert torch.equal(bv[0, :5], vv[:5]) and (bv[0, 5:] == 0).all()
    pool.copy_block(4, 0)
    assert torch.equal(torch.stack(pool.read_block_kv(0, layer)),
                       torch.stack(pool.read_block_kv(4, layer)))
    cache = pool.layer(layer)
    assert isinstance(cache, KVCache8) and cache.codes.dtype == fmt
    assert torch.equal(cache.dequantize()[1, 0, 3].half(), kk[19])
    with pytest.raises(IndexError):
        pool.write_kv(6, 0, k[0], v[0], layer)
    with pytest.raises(IndexError):
        pool.read_kv(0, 16, layer)


def test_half_the_memory():
    small, big = _pool(torch.int8, 2), CUDAMemoryPool(6, 16, 2, 64, torch.float16, "cpu", 2)
    assert small.get_memory_mb() == big.get_memory_mb() * (64 + 4) / 128
    assert small.utilisation_snapshot()["num_blocks"] == 6 and "CUDACache8Pool" in repr(small)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layers", [None, 2])
def test_swapped_blocks_come_back(layers, fmt):
    pool = _pool(fmt, layers)
    g = torch.Generator().manual_seed(2)
    for block in (1, 3, 5):
        k, v = torch.randn((2, 2, 64), generator=g)
        pool.write_kv(block, block, k, v, 0 if layers is None else 1)
    before = [t.clone() for t in pool.tensors()]
    swap = SwapSpace(pool, 4)
    swap.copy_out([5, 1], [0, 2])
    for t in pool.tensors():
        t.zero_()
    swap.copy_in([2, 0], [3, 4])
    dim = 0 if layers is None else 1
    for t, b in zip(pool.tensors(), before):
        assert torch.equal(t.select(dim, 3), b.select(dim, 1))
        assert torch.equal(t.select(dim, 4), b.select(dim, 5))
        assert (t.select(dim, 1) == 0).all()
