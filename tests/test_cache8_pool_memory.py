"""Memory of the 8-bit pool and of the 16-bit pages it hands out (CPU)."""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200 import kernels as K
from vllm_mps_b200.memory.cuda_memory_pool import CUDACache8Pool


@pytest.mark.parametrize("layers", [None, 1, 5])
def test_sized_to_free_memory_with_the_pages_it_hands_out(monkeypatch, layers):
    free = 3 << 20
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (free, 2 * free))
    pool = CUDACache8Pool.from_free_memory(16, 2, 64, torch.float16, "cpu", layers, fraction=0.5)
    monkeypatch.setattr(K, "read_cache8", lambda cache, bt, lens, pages, dst: pages)
    pages = pool.read_back(0, None, None, None, pool.num_blocks)
    held = sum(t.numel() * t.element_size() for t in (*pool.tensors(), pages))
    assert held <= free // 2 < held * (pool.num_blocks + 1) / pool.num_blocks
    few = CUDACache8Pool.from_free_memory(16, 2, 64, torch.float16, "cpu", layers, max_blocks=3)
    assert few.num_blocks == 3 and few.dtype == torch.float16
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (1000, 2000))
    with pytest.raises(MemoryError):
        CUDACache8Pool.from_free_memory(16, 2, 64, torch.float16, "cpu", layers)


def test_pages_handed_out_are_kept_and_grow(monkeypatch):
    pool = CUDACache8Pool(40, 16, 2, 64, torch.bfloat16, "cpu", 2)
    monkeypatch.setattr(K, "read_cache8", lambda cache, bt, lens, pages, dst: pages)
    sizes, last = [], None
    for n in (0, 3, 3, 5, 4, 7, 11, 30, 40, 50):
        pages = pool.read_back(1, None, None, None, n)
        assert pages.dtype == torch.bfloat16 and pages.shape[0] >= n
        assert last is None or pages.shape[0] >= last.shape[0]
        last = pages
        sizes.append(pages.shape[0])
    assert sizes == [1, 3, 3, 6, 6, 12, 12, 30, 40, 50]
