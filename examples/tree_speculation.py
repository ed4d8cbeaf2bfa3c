"""Greedy decoding with a drafted tree: tokens per pass and time against plain decoding.

Builds a random-weight Llama of the given size (there is nothing to download),
decodes a few prompts with the engine and with ``TreeDecoder`` and prints how
many tokens a round decided, and how many it would have to for the same time.
Random weights have no structure a drafter could exploit beyond rounding, so
real checkpoints accept more; but a drafted level costs about as much as a plain
step here, and at none of the sizes tried was the break-even reached.

    python examples/tree_speculation.py [--layers 8] [--hidden 2048] [--batch 4] [--tokens 64]
"""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--widths", type=int, nargs="+", default=[3, 2, 1])
    a = ap.parse_args()

    from transformers import LlamaConfig, LlamaForCausalLM

    from vllm_mps_b200.core.sequence import SamplingParams
    from vllm_mps_b200.engine.llm_engine import LLMEngine
    from vllm_mps_b200.engine.tree_decoder import TreeDecoder

    cfg = LlamaConfig(hidden_size=a.hidden, intermediate_size=a.hidden * 11 // 4 // 64 * 64,
                      num_hidden_layers=a.layers, num_attention_heads=a.hidden // 64,
                      num_key_value_heads=max(1, a.hidden // 512), vocab_size=32000,
                      max_position_embeddings=2048, tie_word_embeddings=False)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).half().eval()
    engine = LLMEngine.from_model(model, num_gpu_blocks=1024, max_batch_size=a.batch,
                                  mode="physical", dtype=torch.float16, device="cuda")
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 32000, (32 + 7 * i,), generator=g).tolist() for i in range(a.batch)]

    def timed(fn):
        fn()
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = fn()
        torch.cuda.synchronize()
        return out, time.perf_counter() - t

    def plain():
        ids = [engine.add_request(p, SamplingParams(temperature=0.0, max_tokens=a.tokens))
               for p in prompts]
        while not engine.is_finished():
            engine.step()
        return [engine.get_output(i).token_ids for i in ids]

    want, t0 = timed(plain)
    decoder = TreeDecoder(engine, widths=a.widths)
    got, t1 = timed(lambda: decoder.generate(prompts, a.tokens))
    same = sum(x == y for p, q in zip(want, got) for x, y in zip(p, q))
    per_round = decoder.accepted / max(1, decoder.rounds)
    print(f"engine {t0 * 1e3:.1f} ms, tree of {len(decoder.tree)} nodes {t1 * 1e3:.1f} ms, "
          f"{per_round:.2f} tokens a round (as fast at {per_round * t1 / t0:.2f}), "
          f"{same} of {a.batch * a.tokens} tokens equal")


if __name__ == "__main__":
    main()
