"""Metadata of prefill chunks: tables for pages that are read back, where they are (CPU)."""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200.core.kv_cache_manager import KVCacheManager
from vllm_mps_b200.models.llama_adapter import build_prefill_metadata


def _chunk(lens):
    kv = KVCacheManager(64, 4)
    for sid, n in enumerate(lens):
        kv.allocate(sid)
        kv.append_slots(sid, n)
    return kv


@pytest.mark.parametrize("pieces", [
    [(0, 0, 4), (1, 16, 23), (2, 0, 16)], [(1, 0, 1)], [(2, 15, 2), (0, 4, 1)], [(1, 32, 8), (2, 0, 17)],
])
def test_only_pools_that_are_read_back_have_tables_of_them(pieces):
    kv = _chunk([5, 40, 17])
    plain = build_prefill_metadata(kv, pieces, 16, torch.device("cpu"))
    assert not any(hasattr(plain, name) for name in ("kv_lens", "dst_tensor", "pages"))
    S, rows = len(pieces), sum(n for _, _, n in pieces)
    # One buffer holds what the 16-bit path reads and no more.
    assert plain.bt_tensor.untyped_storage().nbytes() == 4 * (plain.bt_tensor.numel() + 3 * S + 2 * rows)
    meta = build_prefill_metadata(kv, pieces, 16, torch.device("cpu"), True)
    for name in ("bt_tensor", "q_start", "q_lens", "cu_q", "pos_tensor", "slot_mapping"):
        assert torch.equal(getattr(meta, name), getattr(plain, name))
    lens = [a + n for _, a, n in pieces]
    assert meta.kv_lens.tolist() == lens
    pages = [(n + 15) // 16 for n in lens]
    assert meta.pages == sum(pages) and meta.dst_tensor.shape == meta.bt_tensor.shape
    assert [x for i, n in enumerate(pages) for x in meta.dst_tensor[i, :n].tolist()] == list(range(sum(pages)))
    assert all((meta.dst_tensor[i, n:] == 0).all() for i, n in enumerate(pages))
