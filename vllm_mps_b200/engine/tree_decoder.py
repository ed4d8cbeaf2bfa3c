"""Greedy speculative decoding with a drafted tree, on an engine's model and cache.

The drafter is the model itself with 4-bit weights (``kernels.w4_gemm``): it
shares the target's K/V of everything already decided, so it needs no cache of
its own.  One round of every sequence:

1. Draft: the root (the last decided token) and then each level of the tree
   but the last runs through the 4-bit model; every node writes its K/V after
   the context and attends to the context and its ancestors
   (``kernels.paged_tree_attention`` with the level's rows alone); a node's
   children are its ``width`` best next tokens.
2. Check: all nodes run through the 16-bit model in one pass, writing their
   K/V over the drafter's.
3. Commit: ``kernels.commit_tree`` walks the branch the model agrees with and
   moves its K/V, in every layer, to the slots right after the context.

Every round decides at least one token (the model's own choice after the
root), so the output is the greedy one whatever the drafter proposes.  No
counterpart in the reference, which decodes one token per pass.

A round is one CUDA graph per batch bucket: the host packs tables, slots,
positions and roots into one buffer, one copy in, one replay, one copy of the
decided tokens out.  Padding rows are sequences of length 0: they own no slot,
see nothing and commit nothing.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

from vllm_mps_b200 import kernels as K
from vllm_mps_b200.config import BLOCK_SIZE
from vllm_mps_b200.core.draft_tree import DraftTree
from vllm_mps_b200.models.llama_adapter import build_prefill_metadata


class _Weights:
    """The projections of one model: 16-bit or 4-bit, called the same way."""

    def __init__(self, project, gate_up, head):
        self.project = project  # (layer, "qkv" | "o" | "down", x) -> x @ w.T
        self.gate_up = gate_up  # (layer, x) -> silu(x @ Wg.T) * (x @ Wu.T)
        self.head = head        # x -> logits


class TreeDecoder:
    """Tree-drafted greedy decoding over a physical-mode engine of a Llama-family model.

    ``widths[d]`` children per node of level d; the tree has at most 1024
    nodes.  ``group_size``: columns per scale of the 4-bit weights.  The
    engine's pool, block tables and weights are used as they are; sequences
    decoded here have table ids of their own and free them when done.
    """

    def __init__(self, engine, widths=(3, 2, 2), group_size: int = 64) -> None:
        graphs = engine._graphs
        if engine.mode != "physical" or graphs is None or not graphs.fused:
            raise ValueError("TreeDecoder needs a physical-mode engine of a Llama-family model "
                             "(bias-free SiLU-gated layers) with CUDA graphs enabled")
        model = engine.adapter.hf_model
        if model.lm_head.bias is not None or any(
                layer.mlp.down_proj.bias is not None or layer.self_attn.W_O.bias is not None
                for layer in model.model.layers):
            raise ValueError("TreeDecoder needs projections without bias")
        self.engine = engine
        self.tree = DraftTree.from_widths(tuple(widths))
        if len(self.tree) > 1024:
            raise ValueError(f"a tree of {len(self.tree)} nodes (at most 1024)")
        self.widths = tuple(int(w) for w in widths)
        self.device = engine.model_config.device
        self._mask = torch.from_numpy(self.tree.mask()).to(self.device)
        self._parents = torch.from_numpy(self.tree.parents).to(self.device)
        self._target = self._sixteen_bit()
        self._draft = self._four_bit(group_size)
        self._graphs: dict[int, tuple] = {}
        self._pool = None
        self.rounds = 0
        self.accepted = 0

    # ── the two models ───────────────────────────────────────────────────────

    def _sixteen_bit(self) -> _Weights:
        m = self.engine.adapter.hf_model
        gate_up = self.engine._graphs._gate_up

        def weight(i, name):
            layer = m.model.layers[i]
            return {"qkv": layer.self_attn._w_qkv, "o": layer.self_attn.W_O.weight,
                    "down": layer.mlp.down_proj.weight}[name]

        def act(i, x):
            w = gate_up[i]
            if K.decode_gemm_supported(x.shape[0], w.shape[0] // 2, x.shape[1], True):
                return K.decode_gemm(x, w, silu_mul=True)
            return K.silu_mul(torch.matmul(x, w.t()))

        project = m.model.layers[0].self_attn.project
        return _Weights(lambda i, name, x: project(x, weight(i, name)), act,
                        lambda x: project(x, m.lm_head.weight))

    def _four_bit(self, group_size: int) -> _Weights:
        m = self.engine.adapter.hf_model
        gate_up = self.engine._graphs._gate_up
        q = lambda w: K.quantize_w4(w, group_size)  # noqa: E731
        layers = [dict(qkv=q(layer.self_attn._w_qkv), o=q(layer.self_attn.W_O.weight),
                       down=q(layer.mlp.down_proj.weight), gate_up=q(gate_up[i]))
                  for i, layer in enumerate(m.model.layers)]
        head = q(m.lm_head.weight)
        return _Weights(lambda i, name, x: _w4(x, layers[i][name]),
                        lambda i, x: _w4(x, layers[i]["gate_up"], silu_mul=True),
                        lambda x: _w4(x, head))

    # ── one forward pass over the rows of some nodes ─────────────────────────

    def _forward(self, weights: _Weights, tokens: torch.Tensor, meta: dict) -> torch.Tensor:
        """Logits of the rows; their K/V is written and attended to on the way."""
        m = self.engine.adapter.hf_model
        layers = m.model.layers
        pool = self.engine.memory_pool
        first = layers[0].input_layernorm
        res, h = K.embed_rmsnorm(m.model.embed_tokens.weight, first.weight,
                                 first.variance_epsilon, tokens)
        for i, layer in enumerate(layers):
            a = layer.self_attn
            qkv = weights.project(i, "qkv", h)
            nq, nkv = a.n_heads * a.d_k, a.n_kv_heads * a.d_k
            q = K.rope_reshape_and_cache(qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:],
                                         meta["pos"], meta["slots"], a.rotary_emb.inv_freq,
                                         pool.layer(i))
            out = K.paged_tree_attention(q.unflatten(1, (a.n_heads, a.d_k)), pool.layer(i),
                                         meta["bt"], meta["ctx"], meta["lens"], meta["q_lens"],
                                         meta["cu"], meta["mask"], meta["max_q"],
                                         scale=1.0 / math.sqrt(a.d_k))
            attn = weights.project(i, "o", out.flatten(1))
            post = layer.post_attention_layernorm
            K.add_rmsnorm(res, post.weight, post.variance_epsilon, delta=attn, out=h)
            mlp = weights.project(i, "down", weights.gate_up(i, h))
            nxt = layers[i + 1].input_layernorm if i + 1 < len(layers) else m.model.norm
            K.add_rmsnorm(res, nxt.weight, nxt.variance_epsilon, delta=mlp, out=h)
        return weights.head(h)

    # ── a round as a graph ───────────────────────────────────────────────────

    def _passes(self) -> list[np.ndarray]:
        """The nodes of every pass of a round: the drafted levels, then the whole tree."""
        return [self.tree.level(d) for d in range(len(self.widths))] + [np.arange(len(self.tree))]

    def _static(self, Bb: int) -> SimpleNamespace:
        """Buffers of a bucket: [tables Bb x W | contexts | roots | per pass: slots, positions,
        lengths], and what never changes."""
        W, n = self.engine._graphs.max_blocks, len(self.tree)
        passes = self._passes()
        size = Bb * W + 2 * Bb + sum(2 * Bb * len(nodes) + Bb for nodes in passes)
        dev = torch.zeros(size, dtype=torch.int32, device=self.device)
        host = torch.zeros(size, dtype=torch.int32).pin_memory()
        views, at = [], 0

        def take(count):
            nonlocal at
            view = (at, at + count)
            at += count
            return view

        bt, ctx, root = take(Bb * W), take(Bb), take(Bb)
        for nodes in passes:
            views.append((take(Bb * len(nodes)), take(Bb * len(nodes)), take(Bb)))
        cut = lambda v: dev[v[0]:v[1]]  # noqa: E731
        ids = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
        metas = []
        for nodes, (slots, pos, lens) in zip(passes, views):
            q = len(nodes)
            metas.append(dict(
                bt=cut(bt).view(Bb, W), ctx=cut(ctx), slots=cut(slots), pos=cut(pos),
                lens=cut(lens), q_lens=ids([q] * Bb), cu=ids([i * q for i in range(Bb)]), max_q=q,
                mask=self._mask[nodes[0]:nodes[-1] + 1].repeat(Bb, 1)))
        return SimpleNamespace(Bb=Bb, W=W, dev=dev, host=host, passes=passes, views=views, bt=bt,
                               ctx=ctx, root=root, metas=metas, cut=cut,
                               parents=self._parents.repeat(Bb),
                               tokens=torch.zeros((Bb, n), dtype=torch.int32, device=self.device),
                               result=torch.zeros((Bb, n + 2), dtype=torch.int32, device=self.device),
                               landed=torch.zeros((Bb, n + 2), dtype=torch.int32).pin_memory())

    def _body(self, st: SimpleNamespace) -> None:
        """Draft, check and commit on the static buffers."""
        tree, n, tokens = self.tree, len(self.tree), st.tokens
        tokens[:, 0] = st.cut(st.root)
        for d, width in enumerate(self.widths):
            nodes, kids = st.passes[d], tree.level(d + 1)
            rows = tokens[:, nodes[0]:nodes[-1] + 1].flatten().contiguous()
            logits = self._forward(self._draft, rows, st.metas[d])
            tokens[:, kids[0]:kids[-1] + 1] = logits.topk(width, dim=-1).indices.view(st.Bb, -1)
        meta, flat = st.metas[-1], tokens.view(-1)
        target = self._forward(self._target, flat, meta).argmax(-1)
        path, count, nxt = K.commit_tree(self.engine.memory_pool._all, meta["bt"], meta["ctx"],
                                         meta["lens"], meta["cu"], st.parents, flat, target, n)
        st.result[:, :n] = tokens.gather(1, path.clamp(min=0).long())
        st.result[:, n] = count
        st.result[:, n + 1] = nxt

    def _capture(self, Bb: int):
        st = self._static(Bb)
        for _, (slots, _, _) in zip(st.passes, st.views):
            st.cut(slots).fill_(-1)  # the warm-up rows own no slot
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side), torch.no_grad():
            self._body(st)
        torch.cuda.current_stream(self.device).wait_stream(side)
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        if self._pool is None:
            self._pool = torch.cuda.graph_pool_handle()
        with torch.cuda.graph(g, pool=self._pool), torch.no_grad():
            self._body(st)
        return g, st

    def _claim(self, sids: list[int], ctx: list[int]) -> list[int]:
        """How many nodes of the tree each sequence has in this round, with their slots.

        The first of them (a parent comes before its children): all, unless the
        block table ends or the pool is full before.  The roots' slots are there."""
        kv, n = self.engine.kv_cache_manager, len(self.tree)
        limit = self.engine._graphs.max_blocks * BLOCK_SIZE
        keep = []
        for s, c in zip(sids, ctx):
            want = min(n, limit - c)
            room = kv.free_slots_in_last_block(s) + BLOCK_SIZE * kv.get_num_free_gpu_blocks()
            kv.append_slots(s, min(c + want - kv.num_tokens(s), room))
            keep.append(min(want, kv.num_tokens(s) - c))
        return keep

    def _round(self, sids: list[int], last: list[int], ctx: list[int], keep: list[int]):
        """One draft, check and commit of every sequence: (accepted tokens, next token) each.

        ``keep``: the nodes of each sequence's tree.  The rows of the others run along, own no
        slot, and are past the sequence's length for the commit and every other row."""
        kv = self.engine.kv_cache_manager
        n, B = len(self.tree), len(sids)
        Bb = 1
        while Bb < B:
            Bb *= 2
        if Bb not in self._graphs:
            self._graphs[Bb] = self._capture(Bb)
        g, st = self._graphs[Bb]
        h = st.host.numpy()
        h[:] = 0
        bt = h[st.bt[0]:st.bt[1]].reshape(Bb, st.W)
        for i, s in enumerate(sids):
            table = kv.get_block_ids(s)
            bt[i, :len(table)] = table
        host_ctx, kept = np.asarray(ctx, dtype=np.int64), np.asarray(keep, dtype=np.int64)
        nodes = np.arange(n)
        own = nodes < kept[:, None]
        at = np.where(own, host_ctx[:, None] + nodes, 0)
        slots = np.take_along_axis(bt[:B], at // BLOCK_SIZE, 1).astype(np.int64) * BLOCK_SIZE + at % BLOCK_SIZE
        slots[~own] = -1
        h[st.ctx[0]:st.ctx[0] + B] = host_ctx
        h[st.root[0]:st.root[0] + B] = last
        for nodes, (v_slots, v_pos, v_lens) in zip(st.passes, st.views):
            h[v_slots[0]:v_slots[1]] = -1
            rows = B * len(nodes)
            h[v_slots[0]:v_slots[0] + rows] = slots[:, nodes].reshape(-1)
            h[v_pos[0]:v_pos[0] + rows] = (host_ctx[:, None] + self.tree.depths[nodes]).reshape(-1)
            h[v_lens[0]:v_lens[0] + B] = host_ctx + np.minimum(kept, int(nodes[-1]) + 1)
        st.dev.copy_(st.host, non_blocking=True)
        g.replay()
        st.landed.copy_(st.result, non_blocking=True)
        torch.cuda.current_stream(self.device).synchronize()
        out = st.landed.numpy()[:B]
        self.rounds += B
        self.accepted += int(out[:, n].sum())
        return [(row[1:row[n]].tolist(), int(row[n + 1])) for row in out]

    def _prefill(self, sids: list[int], prompts: list[list[int]]) -> None:
        """K/V of every prompt token but the last, in chunks of the engine's row limit."""
        eng = self.engine
        pieces, rows = [], 0

        def flush():
            meta = build_prefill_metadata(eng.kv_cache_manager, [(s, a, n) for s, a, n, _ in pieces],
                                          BLOCK_SIZE, self.device)
            toks = [t for _, a, n, p in pieces for t in p[a:a + n]]
            toks += [0] * (eng._graphs.padded_rows(len(toks)) - len(toks))
            eng._graphs.prefill_rows(torch.tensor(toks, dtype=torch.int32).to(self.device), meta)

        for sid, prompt in zip(sids, prompts):
            start, need = 0, len(prompt) - 1
            while start < need:
                take = min(need - start, eng.max_prefill_rows - rows)
                pieces.append((sid, start, take, prompt))
                start, rows = start + take, rows + take
                if rows == eng.max_prefill_rows:
                    flush()
                    pieces, rows = [], 0
        if pieces:
            flush()

    @torch.no_grad()
    def generate(self, prompts: list[list[int]], max_tokens: int) -> list[list[int]]:
        """``max_tokens`` greedy tokens for each prompt (lists of token ids, none empty).

        Near the end of the block table or with a full pool a round's trees get
        smaller, down to the root alone (a plain step).  Where the pool does not
        hold all sequences, the last ones wait, or give their blocks back and are
        prefilled again later.  A prompt that could never be finished is refused
        before anything runs: ``MemoryError`` if the free blocks do not hold it
        and its tokens, ``ValueError`` if the block table does not.
        """
        if any(len(p) == 0 for p in prompts):
            raise ValueError("every prompt needs at least one token")
        if max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        kv = self.engine.kv_cache_manager
        free, width = kv.get_num_free_gpu_blocks(), self.engine._graphs.max_blocks
        for p in prompts:
            slots = len(p) + max_tokens - 1  # the last token's K/V is never written
            blocks = -(-slots // BLOCK_SIZE)
            if blocks > free:
                raise MemoryError(f"a prompt of {len(p)} tokens and {max_tokens} more need {blocks} "
                                  f"blocks, {free} are free")
            if blocks > width:
                raise ValueError(f"a prompt of {len(p)} tokens and {max_tokens} more need {blocks} "
                                 f"blocks, the model's length allows {width}")
        taken = set(kv.get_all_seq_ids())
        sids, sid = [], -1
        while len(sids) < len(prompts):
            if sid not in taken:
                sids.append(sid)
            sid -= 1
        out = [[] for _ in prompts]
        live, waiting = [], list(range(len(prompts)))
        try:
            while live or waiting:
                fresh = []
                # One that joins others leaves each of them a block to go on with.
                while waiting and (kv.blocks_needed(sids[waiting[0]], len(prompts[waiting[0]] + out[waiting[0]]))
                                   + len(live) <= kv.get_num_free_gpu_blocks() or not live):
                    i = waiting.pop(0)
                    live.append(i)
                    fresh.append(i)
                    kv.allocate(sids[i])
                    kv.append_slots(sids[i], len(prompts[i]) + len(out[i]))
                self._prefill([sids[i] for i in fresh], [prompts[i] + out[i] for i in fresh])
                # A slot for every root; the last sequences make room for the first.
                at = 0
                while at < len(live):
                    i = live[at]
                    short = len(prompts[i]) + len(out[i]) - kv.num_tokens(sids[i])
                    if short > 0 and not kv.can_allocate(sids[i], short):
                        waiting.insert(0, live.pop())
                        kv.free(sids[waiting[0]])
                    else:
                        kv.append_slots(sids[i], short)
                        at += 1
                ids = [sids[i] for i in live]
                last = [(out[i] or prompts[i])[-1] for i in live]
                ctx = [len(prompts[i]) + len(out[i]) - 1 for i in live]
                for i, (path, nxt) in zip(live, self._round(ids, last, ctx, self._claim(ids, ctx))):
                    out[i] += path + [nxt]
                    if len(out[i]) >= max_tokens:
                        kv.free(sids[i])
                live = [i for i in live if len(out[i]) < max_tokens]
            return [o[:max_tokens] for o in out]
        finally:
            for s in sids:
                if kv.has_sequence(s):
                    kv.free(s)


def _w4(x: torch.Tensor, w: K.W4Weight, silu_mul: bool = False) -> torch.Tensor:
    """``w4_gemm`` for any number of rows."""
    if x.shape[0] <= 32:
        return K.w4_gemm(x, w, silu_mul=silu_mul)
    return torch.cat([K.w4_gemm(part, w, silu_mul=silu_mul) for part in x.split(32)])
