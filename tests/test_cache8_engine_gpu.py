"""The engine over an 8-bit cache, and layers with norms of queries and keys.

The reference is the model in fp32 (below, from its weights) whose K and V are
rounded to codes as the cache rounds them.  Bar: every token the engine emits
has a logit within 0.05 of the reference's best one with a 16-bit cache (the
bar of the engine's other fp16 checks, which is set by 2^-11 of activations
along the way), and within 0.1 with an 8-bit one: what the engine stores differs
from the reference's by those same 2^-11, a code is a rounding without bias, so
the codes' difference adds the same once more.
"""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 900, 3], [44], list(range(100, 150)), [7] * 16, list(range(300, 437))]


def _model(norms, seed=3):
    from transformers import LlamaConfig, LlamaForCausalLM
    from transformers.models.llama.modeling_llama import LlamaRMSNorm

    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
                      num_attention_heads=8, num_key_value_heads=2, vocab_size=1000,
                      max_position_embeddings=1024, tie_word_embeddings=False)
    torch.manual_seed(seed)
    model = LlamaForCausalLM(cfg).half().eval()
    if norms:
        for layer in model.model.layers:
            for name in ("q_norm", "k_norm"):
                norm = LlamaRMSNorm(64, eps=1e-5).half()
                norm.weight.data.copy_(1 + 0.3 * torch.randn(64))
                setattr(layer.self_attn, name, norm)
    return model


class _Reference:
    """The model's logits in fp32, K and V rounded to ``fmt``'s codes (None: not)."""

    def __init__(self, model, fmt):
        self.fmt = fmt
        f = lambda t: t.detach().float().cuda()  # noqa: E731
        m = model.model
        self.embed, self.head, self.norm = f(m.embed_tokens.weight), f(model.lm_head.weight), f(m.norm.weight)
        self.eps = m.norm.variance_epsilon
        self.layers = []
        for layer in m.layers:
            a, p = layer.self_attn, layer.mlp
            w = dict(q=a.q_proj, k=a.k_proj, v=a.v_proj, o=a.o_proj, gate=p.gate_proj, up=p.up_proj,
                     down=p.down_proj, n1=layer.input_layernorm, n2=layer.post_attention_layernorm)
            w = {n: f(x.weight) for n, x in w.items()}
            for name in ("q_norm", "k_norm"):
                w[name] = f(getattr(a, name).weight) if hasattr(a, name) else None
            self.layers.append(w)

    def _rms(self, x, w, eps):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w

    def _kept(self, x):
        if self.fmt is None:
            return x
        codes, scales = K.quantize_cache8(x, self.fmt)
        return codes.float() * scales.unsqueeze(-1)

    @torch.no_grad()
    def logits(self, tokens):
        n = len(tokens)
        x = self.embed[torch.tensor(tokens, device="cuda")]
        inv = 1.0 / (10000.0 ** (torch.arange(0, 64, 2, device="cuda").float() / 64))
        angle = torch.arange(n, device="cuda").double().unsqueeze(1) * inv.double()
        cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

        def rope(t):
            lo, hi = t.chunk(2, -1)
            return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

        mask = torch.full((n, n), float("-inf"), device="cuda").triu(1)
        for w in self.layers:
            h = self._rms(x, w["n1"], self.eps)
            q, k, v = (torch.matmul(h, w[c].t()).view(n, -1, 64) for c in "qkv")
            if w["q_norm"] is not None:
                q, k = self._rms(q, w["q_norm"], 1e-5), self._rms(k, w["k_norm"], 1e-5)
            q, k, v = rope(q), self._kept(rope(k)), self._kept(v)
            k, v = k.repeat_interleave(4, 1), v.repeat_interleave(4, 1)
            s = torch.einsum("qhd,khd->hqk", q, k) / 8 + mask
            o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(n, -1)
            x = x + torch.matmul(o, w["o"].t())
            h = self._rms(x, w["n2"], self.eps)
            g = torch.matmul(h, w["gate"].t())
            x = x + torch.matmul(torch.nn.functional.silu(g) * torch.matmul(h, w["up"].t()), w["down"].t())
        return torch.matmul(self._rms(x, self.norm, self.eps), self.head.t())


def _engine(model, **kw):
    from vllm_mps_b200.engine.llm_engine import LLMEngine

    kw = {"num_gpu_blocks": 128, "max_batch_size": 8, "mode": "physical", **kw}
    return LLMEngine.from_model(model, dtype=torch.float16, device="cuda", **kw)


def _generate(eng, prompts, n=24):
    from vllm_mps_b200.core.sequence import SamplingParams

    ids = [eng.add_request(p, SamplingParams(temperature=0.0, max_tokens=n)) for p in prompts]
    for _ in range(2000):
        if eng.is_finished():
            return [eng.get_output(i).token_ids for i in ids]
        eng.step()
    raise AssertionError("the engine does not finish")


def _check_greedy(reference, prompts, outs, bar):
    for p, o in zip(prompts, outs):
        logits = reference.logits(p + o)
        for k, t in enumerate(o):
            row = logits[len(p) - 1 + k]
            assert float(row.max() - row[t]) <= bar, (len(p), k, t)


CACHES = [None, "int8", "fp8"]
FMT = {None: None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("cache", CACHES)
def test_greedy_tokens(cache, norms):
    model = _model(norms)
    reference = _Reference(model, FMT[cache])
    eng = _engine(model, kv_cache=cache)
    outs = _generate(eng, PROMPTS)
    _check_greedy(reference, PROMPTS, outs, 0.05 if cache is None else 0.1)
    layer = eng.adapter.paged_layers[0]
    assert layer.eight_bit == (cache is not None)
    assert layer.fused_step == (cache is None and not norms)


@pytest.mark.parametrize("kw", [dict(cuda_graphs=False), dict(pipeline=True),
                                dict(max_prefill_rows=40), dict(max_prefill_rows=7, cuda_graphs=False)])
def test_other_ways_to_run(kw):
    model = _model(True, seed=4)
    reference = _Reference(model, torch.int8)
    outs = _generate(_engine(model, kv_cache="int8", **kw), PROMPTS)
    _check_greedy(reference, PROMPTS, outs, 0.1)


def test_preempted_blocks_are_swapped():
    """A pool too small for all requests: codes and scales go out and come back.

    (Staggered lengths, as in the 16-bit engine's test: the reference's scheduler
    does not settle where two sequences need a new block in the same step.)
    """
    model = _model(False, seed=5)
    reference = _Reference(model, torch.int8)
    eng = _engine(model, kv_cache="int8", num_gpu_blocks=8, num_cpu_blocks=32, swap=True,
                  max_tokens_per_step=10000)
    prompts = [list(range(3 + 7 * i, 3 + 7 * i + n)) for i, n in enumerate((30, 22, 14))]
    preempted = []
    step = eng.step
    eng.step = lambda: (preempted.append(eng.scheduler.get_num_preempted()), step())
    outs = _generate(eng, prompts, 40)
    assert [len(o) for o in outs] == [40] * 3 and max(preempted) > 0
    _check_greedy(reference, prompts, outs, 0.1)


def test_drafted_trees_with_norms():
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    model = _model(True, seed=6)
    reference = _Reference(model, None)
    eng = _engine(model)
    outs = TreeDecoder(eng, widths=(3, 2)).generate(PROMPTS, 20)
    _check_greedy(reference, PROMPTS, outs, 0.05)


def test_what_is_refused():
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    model = _model(False)
    with pytest.raises(ValueError):
        _engine(model, kv_cache="int4")
    with pytest.raises(ValueError):
        _engine(model, kv_cache="int8", mode="compat")
    with pytest.raises(ValueError):
        TreeDecoder(_engine(model, kv_cache="fp8"))
