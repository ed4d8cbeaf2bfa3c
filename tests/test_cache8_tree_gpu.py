"""Tree attention whose contexts are an 8-bit cache's pages, read back.

The drafts' K and V are written behind the contexts in the 16-bit pages.  The
reference is the formula on the values that the codes stand for, rounded to 16 bits;
its bound is tree attention's own (test_tree_attention_gpu).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_tree_attention_gpu import _call, _case, _check, _reference
from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("n_q, n_kv, D, dtype", [(8, 2, 64, torch.float16), (32, 8, 128, torch.bfloat16)])
def test_drafts_behind_contexts_read_back(cuda_device, n_q, n_kv, D, dtype, fmt):
    seqs = [(137, 8, 8), (0, 5, 5), (16, 20, 20), (1000, 26, 4), (15, 3, 3)]
    c = _case(cuda_device, seqs, n_q, n_kv, D, dtype, seed=3, spare=0.0)
    codes, scales = K.quantize_cache8(c["pool"], fmt)
    cache = K.KVCache8(codes, scales.permute(0, 3, 1, 2).contiguous())
    # The contexts into pages of another pool, numbered through, rubbish where nothing goes.
    pages = [(ctx + n + 15) // 16 for ctx, n, _ in seqs]
    dst = torch.zeros_like(c["bt"])
    for i, at in enumerate(np.cumsum([0] + pages[:-1])):
        dst[i, :pages[i]] = torch.arange(at, at + pages[i])
    pool = torch.full((sum(pages), 2, 16, n_kv, D), float("nan"), dtype=dtype, device=cuda_device)
    K.read_cache8(cache, c["bt"], c["ctx"], pool, dst)
    values = cache.dequantize().to(dtype)
    slots = []
    for i, (ctx, n, _) in enumerate(seqs):
        t = torch.arange(ctx, ctx + n, device=cuda_device)
        src, to = c["bt"][i].long()[t // 16], dst[i].long()[t // 16]
        values[src, :, t % 16] = c["pool"][src, :, t % 16]  # drafts are 16-bit
        slots.append((src, to, t % 16))
    src, to, off = (torch.cat(x) for x in zip(*slots))
    K.rope_reshape_and_cache(None, c["pool"][src, 0, off], c["pool"][src, 1, off], None,
                             (to * 16 + off).int(), None, pool)
    got = _call(K, dict(c, pool=pool, bt=dst))
    assert K.error_word(cuda_device) == 0
    _check(got, _reference(dict(c, pool=values)), dtype, D)
