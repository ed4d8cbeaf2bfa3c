"""Device KV-cache pool in HBM (replaces the reference's memory/mps_memory_pool.py).

Layout is the reference's: ``(num_blocks, 2, block_size, n_kv_heads, head_dim)``,
dim 1 = K (0) / V (1), zero-initialised (mps_memory_pool.py:62-66); this is
the layout the sm_100a kernels read with TMA.  The method set and the
``IndexError`` bounds checks are the reference's (:82-268).  Two modes:

* ``num_layers=None`` -- one pool shared by every layer, as the reference
  engine builds it (engine/llm_engine.py:166-173): every layer writes the
  current token into the same slot, so history slots hold the last layer's
  K/V.  Needed for token-for-token parity with the reference.
* ``num_layers=L`` -- one pool per layer in one allocation
  ``(L, num_blocks, 2, block_size, n_kv, D)``; :meth:`layer` returns layer
  ``i``'s pool (the physically meaningful cache).

``gather_*``/``read_*``/``write_kv`` are the reference's host-side helpers
(torch indexing on the device); the decode hot path does not use them --
the kernels read and write pages in place.

:class:`CUDACache8Pool` keeps 8-bit codes with a scale per token, head and kind
instead (``kernels.KVCache8``), half the memory for the same blocks.
"""

from __future__ import annotations

import logging
from typing import Sequence

import torch

logger = logging.getLogger(__name__)


class CUDAMemoryPool:
    """Fixed-size KV pool tensor on a CUDA device (CPU allowed for host-only use)."""

    def __init__(self, num_blocks: int, block_size: int, n_heads: int, d_k: int,
                 dtype: torch.dtype = torch.float16, device: torch.device | str | None = None,
                 num_layers: int | None = None) -> None:
        if device is None:
            device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_heads = n_heads
        self.d_k = d_k
        self.dtype = dtype
        self.device = torch.device(device)
        self.num_layers = num_layers
        shape = (num_blocks, 2, block_size, n_heads, d_k)
        if num_layers is None:
            self._all = torch.zeros(shape, dtype=dtype, device=self.device)
            self._pool = self._all
        else:
            self._all = torch.zeros((num_layers, *shape), dtype=dtype, device=self.device)
            self._pool = self._all[0]
        logger.info("CUDAMemoryPool: shape=%s, %.2f MB on %s", list(self._all.shape),
                    self.get_memory_mb(), self.device)

    @classmethod
    def from_free_memory(cls, block_size: int, n_heads: int, d_k: int, dtype: torch.dtype,
                         device: torch.device | str, num_layers: int | None = None,
                         fraction: float = 0.85, max_blocks: int | None = None) -> "CUDAMemoryPool":
        """Size the pool to ``fraction`` of the device's free HBM (B200: ~180 GB)."""
        device = torch.device(device)
        free, _ = torch.cuda.mem_get_info(device)
        per_block = 2 * block_size * n_heads * d_k * torch.tensor([], dtype=dtype).element_size()
        per_block *= num_layers or 1
        n = int(free * fraction) // per_block
        if max_blocks is not None:
            n = min(n, max_blocks)
        if n <= 0:
            raise MemoryError("CUDAMemoryPool: no free device memory for a pool")
        return cls(n, block_size, n_heads, d_k, dtype, device, num_layers)

    def layer(self, i: int) -> torch.Tensor:
        """Pool tensor layer ``i`` reads and writes (the shared pool in shared mode)."""
        if self.num_layers is None:
            return self._pool
        return self._all[i]

    # ── single-token access (mps_memory_pool.py:82-135) ──────────────────────

    def write_kv(self, block_id: int, token_pos: int, k: torch.Tensor, v: torch.Tensor,
                 layer: int = 0) -> None:
        self._validate_indices(block_id, token_pos)
        pool = self.layer(layer)
        pool[block_id, 0, token_pos] = k
        pool[block_id, 1, token_pos] = v

    def read_kv(self, block_id: int, token_pos: int, layer: int = 0):
        self._validate_indices(block_id, token_pos)
        pool = self.layer(layer)
        return pool[block_id, 0, token_pos], pool[block_id, 1, token_pos]

    def read_block_kv(self, block_id: int, layer: int = 0):
        self._check_block(block_id, "block_id")
        pool = self.layer(layer)
        return pool[block_id, 0], pool[block_id, 1]

    # ── gathers (mps_memory_pool.py:139-209) ──────────────────────────────────

    def gather_blocks(self, block_ids: Sequence[int], layer: int = 0):
        ids = torch.as_tensor(list(block_ids), dtype=torch.long, device=self.device)
        return self.gather_blocks_tensor(ids, layer)

    def gather_blocks_tensor(self, ids_tensor: torch.Tensor, layer: int = 0):
        pool = self.layer(layer)
        k = pool[ids_tensor, 0].reshape(-1, self.n_heads, self.d_k)
        v = pool[ids_tensor, 1].reshape(-1, self.n_heads, self.d_k)
        return k, v

    def gather_blocks_batched(self, block_tables: list[list[int]], seq_lens: list[int],
                              max_seq_len: int, layer: int = 0):
        """Zero-padded ``(B, max_seq_len, n_heads, d_k)`` gather (kernels.gather_kv)."""
        from vllm_mps_b200.kernels import gather_kv

        B = len(block_tables)
        max_blocks = max(1, max(len(bt) for bt in block_tables))
        bt = torch.zeros(B, max_blocks, dtype=torch.int32)
        for i, row in enumerate(block_tables):
            bt[i, :len(row)] = torch.as_tensor(row, dtype=torch.int32)
        sl = torch.as_tensor(seq_lens, dtype=torch.int32)
        return gather_kv(self.layer(layer), bt.to(self.device), sl.to(self.device), max_seq_len)

    def copy_block(self, src_block_id: int, dst_block_id: int) -> None:
        """Copy a block's K/V (every layer in per-layer mode) (:211-228)."""
        self._check_block(src_block_id, "src_block_id")
        self._check_block(dst_block_id, "dst_block_id")
        if self.num_layers is None:
            self._all[dst_block_id] = self._all[src_block_id]
        else:
            self._all[:, dst_block_id] = self._all[:, src_block_id]

    # ── introspection ────────────────────────────────────────────────────────

    def tensors(self) -> list[torch.Tensor]:
        """Every tensor that holds blocks, blocks in dimension 0 (1 in per-layer mode)."""
        return [self._all]

    def get_memory_mb(self) -> float:
        return sum(t.numel() * t.element_size() for t in self.tensors()) / (1024 * 1024)

    def utilisation_snapshot(self) -> dict:
        return {"device": str(self.device), "shape": list(self._all.shape),
                "memory_mb": self.get_memory_mb(), "num_blocks": self.num_blocks,
                "block_size": self.block_size, "dtype": str(self.dtype),
                "num_layers": self.num_layers}

    def __repr__(self) -> str:
        return (f"CUDAMemoryPool(device={self.device}, shape={list(self._all.shape)}, "
                f"memory={self.get_memory_mb():.2f} MB)")

    def _check_block(self, bid: int, label: str) -> None:
        if bid < 0 or bid >= self.num_blocks:
            raise IndexError(f"CUDAMemoryPool: {label} {bid} out of range "
                             f"(num_blocks={self.num_blocks}).")

    def _validate_indices(self, block_id: int, token_pos: int) -> None:
        """``IndexError`` on a bad block id or slot, like mps_memory_pool.py:257-268."""
        self._check_block(block_id, "block_id")
        if token_pos < 0 or token_pos >= self.block_size:
            raise IndexError(f"CUDAMemoryPool: token_pos {token_pos} out of range "
                             f"(block_size={self.block_size}).")


class CUDACache8Pool(CUDAMemoryPool):
    """The pool as 8-bit codes and fp32 scales; no counterpart in the reference.

    ``code_dtype``: int8 or float8_e4m3fn.  :meth:`layer` returns a
    ``kernels.KVCache8``, which ``norm_rope_and_cache`` writes and
    ``paged_decode_attention_cache8`` reads; :meth:`read_back` hands 16-bit
    pages of some sequences to the attention calls that want them.  The
    host-side helpers take and return values of ``dtype``.
    """

    def __init__(self, num_blocks: int, block_size: int, n_heads: int, d_k: int,
                 dtype: torch.dtype = torch.float16, device: torch.device | str | None = None,
                 num_layers: int | None = None, code_dtype: torch.dtype = torch.int8) -> None:
        if device is None:
            device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        layers = () if num_layers is None else (num_layers,)
        self._scales = torch.zeros((*layers, num_blocks, n_heads, 2, block_size),
                                   dtype=torch.float32, device=device)
        super().__init__(num_blocks, block_size, n_heads, d_k, code_dtype, device, num_layers)
        self.code_dtype = code_dtype
        self.dtype = dtype
        self._scratch: torch.Tensor | None = None

    @classmethod
    def from_free_memory(cls, block_size: int, n_heads: int, d_k: int, dtype: torch.dtype,
                         device: torch.device | str, num_layers: int | None = None,
                         fraction: float = 0.85, max_blocks: int | None = None,
                         code_dtype: torch.dtype = torch.int8) -> "CUDACache8Pool":
        """Size the pool, and the 16-bit pages of one layer that :meth:`read_back` may come to
        hold for its blocks, to ``fraction`` of the device's free memory."""
        device = torch.device(device)
        free, _ = torch.cuda.mem_get_info(device)
        per_block = 2 * block_size * n_heads * ((d_k + 4) * (num_layers or 1) + 2 * d_k)
        n = int(free * fraction) // per_block
        if max_blocks is not None:
            n = min(n, max_blocks)
        if n <= 0:
            raise MemoryError("CUDACache8Pool: no free device memory for a pool")
        return cls(n, block_size, n_heads, d_k, dtype, device, num_layers, code_dtype)

    def layer(self, i: int):
        from vllm_mps_b200.kernels import KVCache8

        if self.num_layers is None:
            return KVCache8(self._all, self._scales)
        return KVCache8(self._all[i], self._scales[i])

    def tensors(self) -> list[torch.Tensor]:
        return [self._all.view(torch.int8), self._scales]

    def read_back(self, layer: int, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  dst_tables: torch.Tensor, pages: int) -> torch.Tensor:
        """16-bit pages of the sequences, at blocks ``dst_tables`` (below ``pages``) of a
        pool that the next call overwrites (calls are ordered by the stream).  It is kept, as
        large as the most pages so far; a pool whose sequences share no blocks has at most
        ``num_blocks``."""
        from vllm_mps_b200.kernels import read_cache8

        held = 0 if self._scratch is None else self._scratch.shape[0]
        if held == 0 or held < pages:
            self._scratch = None  # its memory may serve the larger one
            pages = max(1, pages, min(2 * held, self.num_blocks))
            self._scratch = torch.empty((pages, 2, self.block_size, self.n_heads, self.d_k),
                                        dtype=self.dtype, device=self.device)
        return read_cache8(self.layer(layer), block_tables, seq_lens, self._scratch, dst_tables)

    def write_kv(self, block_id: int, token_pos: int, k: torch.Tensor, v: torch.Tensor,
                 layer: int = 0) -> None:
        from vllm_mps_b200.kernels import quantize_cache8

        self._validate_indices(block_id, token_pos)
        cache = self.layer(layer)
        for kind, x in enumerate((k, v)):
            codes, scales = quantize_cache8(x, self.code_dtype)
            cache.codes[block_id, kind, token_pos] = codes
            cache.scales[block_id, :, kind, token_pos] = scales

    def _values(self, ids, layer: int) -> torch.Tensor:
        """(blocks, 2, block_size, n_heads, d_k) values of some blocks."""
        cache = self.layer(layer)
        codes = cache.codes.view(torch.int8)[ids].view(self.code_dtype).float()
        return (codes * cache.scales[ids].permute(0, 2, 3, 1).unsqueeze(-1)).to(self.dtype)

    def read_kv(self, block_id: int, token_pos: int, layer: int = 0):
        self._validate_indices(block_id, token_pos)
        x = self._values([block_id], layer)[0]
        return x[0, token_pos], x[1, token_pos]

    def read_block_kv(self, block_id: int, layer: int = 0):
        self._check_block(block_id, "block_id")
        x = self._values([block_id], layer)[0]
        return x[0], x[1]

    def gather_blocks_tensor(self, ids_tensor: torch.Tensor, layer: int = 0):
        x = self._values(ids_tensor, layer)
        return (x[:, 0].reshape(-1, self.n_heads, self.d_k),
                x[:, 1].reshape(-1, self.n_heads, self.d_k))

    def gather_blocks_batched(self, block_tables: list[list[int]], seq_lens: list[int],
                              max_seq_len: int, layer: int = 0):
        shape = (len(block_tables), max_seq_len, self.n_heads, self.d_k)
        out = torch.zeros((2, *shape), dtype=self.dtype, device=self.device)
        for i, (table, n) in enumerate(zip(block_tables, seq_lens)):
            n = min(n, max_seq_len)
            if n > 0:
                ids = torch.as_tensor(table[:-(-n // self.block_size)], device=self.device)
                out[0, i, :n], out[1, i, :n] = (t[:n] for t in self.gather_blocks_tensor(ids, layer))
        return out[0], out[1]

    def copy_block(self, src_block_id: int, dst_block_id: int) -> None:
        self._check_block(src_block_id, "src_block_id")
        self._check_block(dst_block_id, "dst_block_id")
        for t in self.tensors():
            if self.num_layers is None:
                t[dst_block_id] = t[src_block_id]
            else:
                t[:, dst_block_id] = t[:, src_block_id]

    def __repr__(self) -> str:
        return super().__repr__().replace("CUDAMemoryPool", "CUDACache8Pool")


class SwapSpace:
    """Pinned host copy of swapped-out blocks: the data half of preemption.

    The reference's swap moves block metadata only and loses the KV data
    (core/kv_cache_manager.py:188, :225) and its CPU pool is never wired in
    (memory/cpu_memory_pool.py).  Attached to a :class:`KVCacheManager`, this
    copies the blocks' K/V (all layers) device->host on swap-out and back on
    swap-in, with one batched copy per direction on the caller's stream.
    """

    def __init__(self, gpu_pool: CUDAMemoryPool, num_cpu_blocks: int) -> None:
        self.gpu_pool = gpu_pool
        self._blk_dim = 0 if gpu_pool.num_layers is None else 1
        self._cpu = []
        for t in gpu_pool.tensors():
            shape = list(t.shape)
            shape[self._blk_dim] = num_cpu_blocks
            host = torch.zeros(shape, dtype=t.dtype)
            self._cpu.append(host.pin_memory() if torch.cuda.is_available() else host)
        self.cpu = self._cpu[0]

    def copy_out(self, gpu_ids: list[int], cpu_ids: list[int]) -> None:
        g = torch.as_tensor(gpu_ids, dtype=torch.long, device=self.gpu_pool.device)
        for t, host in zip(self.gpu_pool.tensors(), self._cpu):
            data = t.index_select(self._blk_dim, g).to("cpu")
            host.index_copy_(self._blk_dim, torch.as_tensor(cpu_ids, dtype=torch.long), data)

    def copy_in(self, cpu_ids: list[int], gpu_ids: list[int]) -> None:
        g = torch.as_tensor(gpu_ids, dtype=torch.long, device=self.gpu_pool.device)
        for t, host in zip(self.gpu_pool.tensors(), self._cpu):
            data = host.index_select(self._blk_dim, torch.as_tensor(cpu_ids, dtype=torch.long))
            t.index_copy_(self._blk_dim, g, data.to(self.gpu_pool.device, non_blocking=True))
