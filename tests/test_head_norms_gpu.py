"""A model of the library's whose own forward normalises queries and keys, in the engine.

Bars and the fp32 reference as in test_cache8_engine_gpu; the reference is held
against the model's own forward in fp32 first (both fp32, sums of up to 1024
products of values below 8 in five places a layer: 1e-3).
"""

from __future__ import annotations

import copy

import pytest
import torch

from test_cache8_engine_gpu import CACHES, FMT, PROMPTS, _check_greedy, _engine, _generate, _Reference

pytestmark = pytest.mark.gpu


def _model():
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(hidden_size=512, intermediate_size=1024, num_hidden_layers=3, head_dim=64,
                      num_attention_heads=8, num_key_value_heads=2, vocab_size=1000, rms_norm_eps=1e-5,
                      max_position_embeddings=1024, tie_word_embeddings=False,
                      attn_implementation="eager")
    torch.manual_seed(8)
    model = Qwen3ForCausalLM(cfg).eval()
    for layer in model.model.layers:
        for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            norm.weight.data.copy_(1 + 0.3 * torch.randn(64))
    return model.half()


@pytest.mark.parametrize("cache", CACHES)
def test_greedy_tokens(cache):
    model = _model()
    tokens = PROMPTS[2]
    full = copy.deepcopy(model).float()
    # (half() has rounded the rotation's frequencies, which the engine works out in fp32.)
    full.model.rotary_emb = type(full.model.rotary_emb)(full.config)
    with torch.no_grad():
        own = full.cuda()(torch.tensor([tokens], device="cuda")).logits[0]
    assert (_Reference(model, None).logits(tokens) - own).abs().max() < 1e-3
    reference = _Reference(model, FMT[cache])
    eng = _engine(model, kv_cache=cache)
    outs = _generate(eng, PROMPTS)
    layer = eng.adapter.paged_layers[0]
    assert layer.q_norm_weight is not None and layer.k_norm_weight is not None and layer.norm_eps == 1e-5
    assert eng._graphs.fused
    _check_greedy(reference, PROMPTS, outs, 0.05 if cache is None else 0.1)
