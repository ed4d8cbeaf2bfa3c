"""Which sequences a tree-drafted round holds and how large their trees are (no GPU).

The model is a stand-in that knows every position's token and accepts a random
branch of what was drafted; tables and slots are the real ones.
"""

from __future__ import annotations

import random
from types import SimpleNamespace

import pytest

from vllm_mps_b200.config import BLOCK_SIZE
from vllm_mps_b200.core.draft_tree import DraftTree
from vllm_mps_b200.core.kv_cache_manager import KVCacheManager
from vllm_mps_b200.engine.tree_decoder import TreeDecoder


def _token(prompt, position):
    return (prompt * 7919 + position * 31) % 997


class _Decoder(TreeDecoder):
    def __init__(self, blocks, width, widths, seed=0):
        self.engine = SimpleNamespace(kv_cache_manager=KVCacheManager(blocks, 1),
                                      _graphs=SimpleNamespace(max_blocks=width))
        self.tree = DraftTree.from_widths(widths)
        self.rng = random.Random(seed)
        self.sizes, self.batches, self.prefilled = [], [], 0
        self.written = {}  # K/V per sequence: how many tokens

    def _prefill(self, sids, prompts):
        for s, p in zip(sids, prompts):
            self.prefilled += 1
            self.written[s] = len(p) - 1

    def _round(self, sids, last, ctx, keep):
        kv = self.engine.kv_cache_manager
        self.batches.append(len(sids))
        self.sizes += keep
        blocks = [b for s in sids for b in kv.get_block_ids(s).tolist()]
        assert len(set(blocks)) == len(blocks)
        out = []
        for s, token, c, k in zip(sids, last, ctx, keep):
            assert 1 <= k <= len(self.tree)
            assert kv.num_tokens(s) >= c + k  # every node has a slot
            assert len(kv.get_block_ids(s)) <= self.engine._graphs.max_blocks
            assert self.written[s] == c       # and the context has its K/V
            prompt = self.which[s]
            assert token == _token(prompt, c)
            deepest = int(self.tree.depths[:k].max())
            count = self.rng.randint(1, deepest + 1)
            self.written[s] = c + count
            out.append(([_token(prompt, c + j) for j in range(1, count)], _token(prompt, c + count)))
        return out

    def run(self, lengths, max_tokens):
        self.which = {-1 - i: i for i in range(len(lengths))}
        prompts = [[_token(i, t) for t in range(n)] for i, n in enumerate(lengths)]
        out = self.generate(prompts, max_tokens)
        for i, (n, o) in enumerate(zip(lengths, out)):
            assert o == [_token(i, n + t) for t in range(max_tokens)]
        kv = self.engine.kv_cache_manager
        assert kv.get_num_free_gpu_blocks() == kv.gpu_allocator.total_blocks
        assert not kv.get_all_seq_ids()
        return self


@pytest.mark.parametrize("widths", [(1,), (3, 2, 2), (4, 4, 4)])
def test_up_to_the_last_slot_of_the_table(widths):
    """Prompt and tokens that fill the table: trees shrink instead of failing."""
    width = 10
    for prompt in (1, 3, 100, 140, 159, 160):
        d = _Decoder(100, width, widths, seed=prompt).run([prompt, 1], width * BLOCK_SIZE - prompt + 1)
        assert min(d.sizes) >= 1
    assert min(d.sizes) == 1 and max(d.sizes) == len(d.tree)


def test_a_full_pool_makes_sequences_wait_not_fail():
    rng = random.Random(5)
    for case in range(60):
        lengths = [rng.randint(1, 90) for _ in range(rng.randint(2, 9))]
        tokens = rng.randint(1, 70)
        least = -(-(max(lengths) + tokens - 1) // BLOCK_SIZE)
        _Decoder(least + rng.randint(0, 6), 40, (3, 2, 2), seed=case).run(lengths, tokens)


def test_with_room_for_all_nothing_waits():
    d = _Decoder(200, 40, (3, 2, 2)).run([20, 31, 7, 64], 40)
    assert d.batches[0] == 4 and d.prefilled == 4
    assert set(d.sizes) == {len(d.tree)}


def test_impossible_requests_are_refused_before_anything_runs():
    d = _Decoder(10, 6, (2,))
    for lengths, tokens, error in (([3, 200], 4, MemoryError), ([3, 90], 8, ValueError)):
        with pytest.raises(error):
            d.run(lengths, tokens)
        assert d.prefilled == 0 and not d.batches
        assert d.engine.kv_cache_manager.get_num_free_gpu_blocks() == 10
    d.run([3, 90], 7)
