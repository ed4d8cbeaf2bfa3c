"""Tree-drafted greedy decoding end to end: the tokens are the model's own greedy ones.

Every emitted token is checked against the model's fp32 forward over the
prefix that was emitted before it: its logit is within 0.05 of the best one
(the bar of the engine's other fp16 checks).  A drafter that proposes nothing
useful and one that is the model itself must both pass; the second decides
whole branches a round.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from transformers import LlamaConfig, LlamaForCausalLM

    from vllm_mps_b200.engine.llm_engine import LLMEngine

    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
                      num_attention_heads=8, num_key_value_heads=2, vocab_size=1000,
                      max_position_embeddings=1024, tie_word_embeddings=False)
    torch.manual_seed(3)
    model = LlamaForCausalLM(cfg).half().eval()
    reference = LlamaForCausalLM(cfg)
    reference.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    eng = LLMEngine.from_model(model, num_gpu_blocks=128, max_batch_size=4, mode="physical",
                               dtype=torch.float16, device="cuda")
    return eng, reference.float().cuda().eval()


PROMPTS = [[5, 17, 900, 3], [44], list(range(100, 150)), [7] * 16]


def _check_greedy(reference, prompts, outs):
    with torch.no_grad():
        for p, o in zip(prompts, outs):
            logits = reference(torch.tensor([p + o], device="cuda")).logits[0]
            for k, t in enumerate(o):
                row = logits[len(p) - 1 + k]
                assert float(row.max() - row[t]) <= 0.05, (k, t)


@pytest.mark.parametrize("widths", [(1,), (3, 2), (2, 2, 2), (4, 1, 1, 1)])
def test_tokens_are_greedy(engine, widths):
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, reference = engine
    free = eng.kv_cache_manager.get_num_free_gpu_blocks()
    dec = TreeDecoder(eng, widths=widths, group_size=128)
    outs = dec.generate(PROMPTS, 24)
    assert [len(o) for o in outs] == [24] * 4
    _check_greedy(reference, PROMPTS, outs)
    assert eng.kv_cache_manager.get_num_free_gpu_blocks() == free  # every table was freed
    assert dec.rounds <= dec.accepted <= dec.rounds * (dec.tree.max_depth + 1)


def test_a_perfect_drafter_decides_whole_branches(engine):
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, reference = engine
    dec = TreeDecoder(eng, widths=(2, 1, 1))
    dec._draft = dec._target
    outs = dec.generate(PROMPTS[:2], 32)
    _check_greedy(reference, PROMPTS[:2], outs)
    assert dec.accepted / dec.rounds > 3.0  # of at most 4


def test_a_useless_drafter_still_decides_greedily(engine):
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, reference = engine
    dec = TreeDecoder(eng, widths=(2, 2))
    head = dec._draft.head
    dec._draft.head = lambda x: -head(x)  # the least likely tokens
    outs = dec.generate(PROMPTS, 8)
    _check_greedy(reference, PROMPTS, outs)
    assert dec.accepted / dec.rounds < 1.5


def test_refusals(engine):
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, _ = engine
    with pytest.raises(ValueError):
        TreeDecoder(eng, widths=(4, 4, 4, 4, 4))
    dec = TreeDecoder(eng, widths=(2,))
    with pytest.raises(ValueError):
        dec.generate([[]], 4)
    with pytest.raises(ValueError):
        dec.generate([[1]], 0)
    free = eng.kv_cache_manager.get_num_free_gpu_blocks()
    with pytest.raises(MemoryError):
        dec.generate([[1] * (16 * 200)], 4)
    assert eng.kv_cache_manager.get_num_free_gpu_blocks() == free


@pytest.mark.parametrize("widths", [(3, 2, 2), (4, 4, 4)])
def test_up_to_the_models_length(engine, widths):
    """Prompt and tokens fill the model's length, the table holds less than a whole tree more."""
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, reference = engine
    g = torch.Generator().manual_seed(8)
    long = torch.randint(0, 1000, (990,), generator=g).tolist()
    dec = TreeDecoder(eng, widths=widths)
    outs = dec.generate([long, [3, 4]], 34)  # 1024 tokens
    assert [len(o) for o in outs] == [34, 34]
    _check_greedy(reference, [long, [3, 4]], outs)
    # One sequence to the table's last slot: at the end the tree is the root alone.
    slots = eng._graphs.max_blocks * 16
    short = long[:slots - 40 - 24 + 1]
    outs = dec.generate([short + [9] * 40], 24)
    _check_greedy(reference, [short + [9] * 40], outs)
    with pytest.raises(ValueError):
        dec.generate([long], slots - 990 + 2)


def test_a_pool_that_does_not_hold_all_sequences(engine):
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    eng, reference = engine
    free = eng.kv_cache_manager.get_num_free_gpu_blocks()
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, 1000, (480 + i,), generator=g).tolist() for i in range(5)]
    dec = TreeDecoder(eng)
    outs = dec.generate(prompts, 60)  # 5 x 540 tokens in 2048 slots
    assert [len(o) for o in outs] == [60] * 5
    _check_greedy(reference, prompts, outs)
    assert eng.kv_cache_manager.get_num_free_gpu_blocks() == free
