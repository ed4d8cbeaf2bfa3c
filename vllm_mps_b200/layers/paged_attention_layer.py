"""Drop-in replacement for HuggingFace ``LlamaAttention`` backed by the paged pool.

Same interface as the reference's layers/paged_attention_layer.py:26-391:
``from_llama_layer`` clones the q/k/v/o projections, ``forward(hidden_states,
**kwargs) -> (out, None)`` ignores HF's RoPE and mask and reads per-step
metadata from ``models.llama_adapter._batch_context``, ``set_context`` feeds
the single-token path, ``evict_sequence`` drops per-sequence caches.

The step between the projections -- RoPE on Q/K, the K/V write into the
sequence's slot, the paged gather, GQA and the softmax attention, which the
reference runs as per-sequence Python loops (:275-359) or as a Metal shader
-- is one call into the sm_100a kernel (``kernels.paged_decode_step``).  Q, K
and V come from one fused projection GEMM and are passed as strided slices
of its output, so nothing is copied or materialised.  There is no CPU path.

Layers with norms of queries and keys per head (``q_norm``/``k_norm`` modules
of head_dim weights) and pools of 8-bit codes take two kernels for the step:
``kernels.norm_rope_and_cache``, then the attention over what it wrote.
"""

from __future__ import annotations

import logging
import math

import torch
import torch.nn as nn

from vllm_mps_b200.config import BLOCK_SIZE
from vllm_mps_b200.core.kv_cache_manager import KVCacheManager
from vllm_mps_b200.core.model_config import ModelConfig
from vllm_mps_b200.layers.rotary_embedding import RotaryEmbedding

logger = logging.getLogger(__name__)


class PagedAttentionLayer(nn.Module):
    """Attention layer that writes and reads K/V through the paged pool."""

    def __init__(self, layer_idx: int, model_config: ModelConfig, kv_cache_manager: KVCacheManager,
                 memory_pool, W_Q: nn.Linear, W_K: nn.Linear, W_V: nn.Linear, W_O: nn.Linear,
                 rotary_emb: RotaryEmbedding, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, norm_eps: float = 1e-6) -> None:
        super().__init__()
        self.layer_idx = layer_idx
        self.model_config = model_config
        self.kv_cache_manager = kv_cache_manager
        self.memory_pool = memory_pool
        self.W_Q, self.W_K, self.W_V, self.W_O = W_Q, W_K, W_V, W_O
        self.rotary_emb = rotary_emb
        self.n_heads = model_config.n_heads
        self.n_kv_heads = model_config.n_kv_heads
        self.d_k = model_config.d_k
        self.d_model = model_config.d_model
        self.block_size = BLOCK_SIZE
        self._current_seq_id: int | None = None
        self._current_position: int | None = None
        self.timer = None
        self._block_ids_cache: dict[int, tuple[tuple[int, ...], torch.Tensor]] = {}
        # One GEMM for Q, K and V: rows [W_Q; W_K; W_V].
        self.register_buffer("_w_qkv", torch.cat([W_Q.weight, W_K.weight, W_V.weight], 0).detach(),
                             persistent=False)
        # Norms of each head of q and k: weights (head_dim,), or None.
        self.register_buffer("q_norm_weight", q_norm, persistent=False)
        self.register_buffer("k_norm_weight", k_norm, persistent=False)
        self.norm_eps = norm_eps
        self._workspace = None

    @classmethod
    def from_llama_layer(cls, layer, layer_idx: int, model_config: ModelConfig,
                         kv_cache_manager: KVCacheManager, memory_pool) -> "PagedAttentionLayer":
        """Build from a HuggingFace ``LlamaAttention``; weights are cloned (:91-148)."""
        dev, dt = model_config.device, model_config.dtype
        n_q, n_kv, D, d = model_config.n_heads, model_config.n_kv_heads, model_config.d_k, model_config.d_model

        def lin(src, out_f, in_f):
            m = nn.Linear(in_f, out_f, bias=False, device=dev, dtype=dt)
            m.weight.data.copy_(src.weight.data.to(device=dev, dtype=dt))
            return m

        if isinstance(layer, PagedAttentionLayer):  # a model already attached to an engine
            srcs = (layer.W_Q, layer.W_K, layer.W_V, layer.W_O)
        else:
            srcs = (layer.q_proj, layer.k_proj, layer.v_proj, layer.o_proj)
        W_Q = lin(srcs[0], n_q * D, d)
        W_K = lin(srcs[1], n_kv * D, d)
        W_V = lin(srcs[2], n_kv * D, d)
        W_O = lin(srcs[3], d, n_q * D)
        rot = RotaryEmbedding(D, model_config.max_seq_len, model_config.rope_theta, dev)
        q_norm, k_norm, eps = cls._head_norms(layer, D)
        on = lambda w: None if w is None else w.detach().to(device=dev, dtype=dt).contiguous()  # noqa: E731
        return cls(layer_idx, model_config, kv_cache_manager, memory_pool, W_Q, W_K, W_V, W_O, rot,
                   on(q_norm), on(k_norm), eps)

    @classmethod
    def _head_norms(cls, layer, d: int):
        """(q weight, k weight, eps) of an attention module's norms over each head, if it has them.

        Only norms that the kernels compute are taken; a layer with others is refused.
        """
        if isinstance(layer, PagedAttentionLayer):
            return layer.q_norm_weight, layer.k_norm_weight, layer.norm_eps
        for name, module in layer.named_children():
            if "norm" in name and name not in ("q_norm", "k_norm") and not isinstance(module, nn.Identity):
                raise NotImplementedError(f"attention with {name} ({type(module).__name__}): norms of "
                                          "queries and keys are q_norm and k_norm")
        q, k = (cls._rms_norm(getattr(layer, name, None), name, d) for name in ("q_norm", "k_norm"))
        if q and k and q[1] != k[1]:
            raise NotImplementedError(f"q_norm and k_norm with different eps ({q[1]:g}, {k[1]:g})")
        return q and q[0], k and k[0], (q or k or (None, 1e-6))[1]

    @staticmethod
    def _rms_norm(module, name: str, d: int):
        """(weight, eps) of an RMS norm over ``d`` values, by what the module computes: some
        modules under these names take off a mean, multiply by 1 + weight or span all heads."""
        if module is None or isinstance(module, nn.Identity):
            return None
        weight = getattr(module, "weight", None)
        eps = getattr(module, "variance_epsilon", getattr(module, "eps", None))
        eps = torch.finfo(torch.float32).eps if eps is None else float(eps)
        plain = weight is not None and weight.numel() == d
        if plain:
            # Rows with a mean, of sizes 1, 30 and that at which eps is half of the sum.
            with torch.no_grad():
                x = 0.5 + torch.randn((3, d), generator=torch.Generator().manual_seed(0))
                x *= torch.tensor([[1.0], [30.0], [max(eps, 1e-8) ** 0.5]])
                x = x.to(weight)
                want = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + eps)
                want *= weight.float().flatten()
                try:
                    got = module(x.view(1, 3, 1, d)).view(3, d).float()
                except Exception:  # made for another shape
                    plain = False
                else:
                    # (The module's own roundings, one or two.)
                    off = 2 * torch.finfo(weight.dtype).eps
                    plain = bool(((got - want).abs() <= off * want.abs() + 1e-6).all())
        if not plain:
            raise NotImplementedError(f"attention whose {name} ({type(module).__name__}) is not "
                                      f"x * weight / sqrt(mean(x^2) + eps) over a head's {d} values")
        return weight, eps

    # ── forward ─────────────────────────────────────────────────────────────

    def forward(self, hidden_states: torch.Tensor, **kwargs):
        from vllm_mps_b200.models.llama_adapter import _batch_context

        if getattr(_batch_context, "is_batch", False):
            return self._forward_batch(hidden_states, _batch_context.seq_ids,
                                       _batch_context.positions, _batch_context.seq_lens)
        return self._forward_single(hidden_states)

    def _pool(self):
        """This layer's pool tensor, or its ``KVCache8``."""
        return self.memory_pool.layer(self.layer_idx)

    @property
    def eight_bit(self) -> bool:
        """Whether the pool holds 8-bit codes."""
        return hasattr(self.memory_pool, "code_dtype")

    @property
    def fused_step(self) -> bool:
        """Whether a decode step's rotation, write and attention are one kernel."""
        return not (self.eight_bit or self.q_norm_weight is not None
                    or self.k_norm_weight is not None)

    def store(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
              positions: torch.Tensor, slot_mapping: torch.Tensor,
              in_place: bool = True) -> torch.Tensor | None:
        """Norms and rotation of q and k; k and v into their slots.  Returns q, rotated in
        its place or (layers without the fused step) in a tensor of its own."""
        from vllm_mps_b200.kernels import norm_rope_and_cache, rope_reshape_and_cache

        if self.fused_step:
            return rope_reshape_and_cache(q, k, v, positions, slot_mapping,
                                          self.rotary_emb.inv_freq, self._pool())
        return norm_rope_and_cache(q, k, v, positions, slot_mapping, self.rotary_emb.inv_freq,
                                   self._pool(), self.q_norm_weight, self.k_norm_weight,
                                   self.norm_eps, q_out=q if in_place else None)

    def _workspace_buf(self):
        if self._workspace is None:
            from vllm_mps_b200.kernels import DecodeWorkspace

            self._workspace = DecodeWorkspace()
        return self._workspace

    @staticmethod
    def project(x2d: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        """``x2d @ w.T``: the decode GEMM kernel at decode batch sizes (M <= 8,
        weight streaming, chained to its neighbours with programmatic dependent
        launch), cuBLAS for everything else."""
        from vllm_mps_b200 import kernels as K

        if (x2d.is_cuda and x2d.stride(1) == 1 and x2d.stride(0) % 8 == 0
                and x2d.data_ptr() % 16 == 0 and w.is_contiguous() and w.data_ptr() % 16 == 0
                and K.decode_gemm_supported(x2d.shape[0], w.shape[0], w.shape[1])):
            return K.decode_gemm(x2d, w)
        return torch.matmul(x2d, w.t())

    def _attend(self, hidden_states: torch.Tensor, meta) -> torch.Tensor:
        """Fused QKV GEMM -> one decode-step kernel -> W_O, for (B, 1, d_model)."""
        from vllm_mps_b200.kernels import (paged_decode_attention, paged_decode_attention_cache8,
                                           paged_decode_step)

        B = hidden_states.shape[0]
        n_q, n_kv, D = self.n_heads, self.n_kv_heads, self.d_k
        qkv = self.project(hidden_states.reshape(B, self.d_model), self._w_qkv)
        q = qkv[:, : n_q * D].view(B, n_q, D)
        k = qkv[:, n_q * D: (n_q + n_kv) * D]
        v = qkv[:, (n_q + n_kv) * D:]
        if self.fused_step:
            out = paged_decode_step(q, k, v, meta.pos_tensor, meta.slot_mapping,
                                    self.rotary_emb.inv_freq, self._pool(), meta.bt_tensor,
                                    meta.sl_tensor, scale=1.0 / math.sqrt(D),
                                    workspace=self._workspace_buf())
        else:
            q = self.store(q, k, v, meta.pos_tensor, meta.slot_mapping, in_place=False)
            if self.eight_bit:
                out = paged_decode_attention_cache8(q, self._pool(), meta.bt_tensor, meta.sl_tensor,
                                                    workspace=self._workspace_buf())
            else:
                out = paged_decode_attention(q, self._pool(), meta.bt_tensor, meta.sl_tensor,
                                             workspace=self._workspace_buf())
        if self.W_O.bias is None:
            return self.project(out.view(B, n_q * D), self.W_O.weight).view(B, 1, -1)
        return self.W_O(out.view(B, 1, n_q * D))

    def _prefill_rows(self, hidden_states: torch.Tensor, meta) -> torch.Tensor:
        """Prompt rows of a prefill chunk: kernel 1 writes every row's K/V, kernel 3 attends.

        Kernel 1 rotates q in place inside the fused QKV output and writes the
        rotated K and V of all rows into their slots; kernel 3 (tcgen05 causal
        prefill) then computes every row against its sequence's slots
        ``0..position`` -- the result of the reference's token-by-token
        single-token path (:175-241) for the whole chunk at once.  Over 8-bit
        codes the chunk's sequences are read back into 16-bit pages first, so
        a row attends to the values that later steps will read.

        ``hidden_states`` may carry padding rows after the chunk's
        ``meta.rows`` rows (a caller that rounds the GEMMs' row count): the
        projections run on every row, kernels 1 and 3 on the chunk's rows
        only, and the padding rows of the result are not meaningful.
        """
        from vllm_mps_b200.kernels import paged_prefill_attention

        B = hidden_states.shape[0]
        R = meta.rows
        n_q, n_kv, D = self.n_heads, self.n_kv_heads, self.d_k
        qkv = torch.matmul(hidden_states.reshape(B, self.d_model), self._w_qkv.t())
        q = qkv[:R, : n_q * D]
        k = qkv[:R, n_q * D: (n_q + n_kv) * D]
        v = qkv[:R, (n_q + n_kv) * D:]
        self.store(q, k, v, meta.pos_tensor, meta.slot_mapping)
        pool, tables = self._pool(), meta.bt_tensor
        if self.eight_bit:
            pool, tables = self.memory_pool.read_back(self.layer_idx, meta.bt_tensor, meta.kv_lens,
                                                      meta.dst_tensor, meta.pages), meta.dst_tensor
        out = torch.empty((B, n_q * D), dtype=qkv.dtype, device=qkv.device)
        if B > R:
            out[R:].zero_()
        paged_prefill_attention(q.view(R, n_q, D), pool, tables, meta.q_start, meta.q_lens,
                                meta.cu_q, meta.max_q_len, scale=1.0 / math.sqrt(D),
                                out=out[:R].view(R, n_q, D))
        return self.W_O(out.view(B, 1, n_q * D))

    def _write_kv_rows(self, hidden_states: torch.Tensor, meta) -> None:
        """Only the K/V half of :meth:`_prefill_rows`: the K and V projections
        and kernel 1's write of every row's rotated K and V (no query, no
        attention).  The last layer of a prefill needs nothing more: no later
        layer reads its output."""
        B, R = hidden_states.shape[0], meta.rows
        n_q, n_kv, D = self.n_heads, self.n_kv_heads, self.d_k
        kv = torch.matmul(hidden_states.reshape(B, self.d_model), self._w_qkv[n_q * D:].t())
        self.store(None, kv[:R, : n_kv * D], kv[:R, n_kv * D:], meta.pos_tensor,
                   meta.slot_mapping)

    def _forward_batch(self, hidden_states: torch.Tensor, seq_ids: list[int],
                       positions: list[int], seq_lens: list[int]):
        """Batched decode, one token per sequence (:245-364); prompt rows in prefill."""
        from vllm_mps_b200.models.llama_adapter import _batch_context

        if getattr(_batch_context, "prefill", False):
            return (self._prefill_rows(hidden_states, _batch_context.prefill_meta), None)
        return (self._attend(hidden_states, _batch_context), None)

    def _forward_single(self, hidden_states: torch.Tensor):
        """Single token at ``set_context``'s (seq_id, position) (:175-241)."""
        from vllm_mps_b200.models.llama_adapter import build_step_metadata

        seq_id, pos = self._current_seq_id, self._current_position
        if seq_id is None or pos is None:
            raise RuntimeError("PagedAttentionLayer: seq_id/position_id not set. "
                               "Call set_context() before forward.")
        meta = build_step_metadata(self.kv_cache_manager, [seq_id], [pos], [pos + 1],
                                   self.block_size, hidden_states.device)
        return (self._attend(hidden_states, meta), None)

    def set_context(self, seq_id: int, position_id: int) -> None:
        self._current_seq_id = seq_id
        self._current_position = position_id

    def _get_cached_ids_tensor(self, seq_id: int, block_ids: list[int]) -> torch.Tensor:
        """Per-sequence block-id tensor cache, rebuilt only when the table grows (:375-387)."""
        t = tuple(block_ids)
        cached = self._block_ids_cache.get(seq_id)
        if cached is None or cached[0] != t:
            tensor = torch.tensor(block_ids, dtype=torch.long, device=self.memory_pool.device)
            self._block_ids_cache[seq_id] = (t, tensor)
            return tensor
        return cached[1]

    def evict_sequence(self, seq_id: int) -> None:
        self._block_ids_cache.pop(seq_id, None)
