"""Norms of queries and keys that an attention layer takes over, and those it refuses (CPU)."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from vllm_mps_b200.layers.paged_attention_layer import PagedAttentionLayer

D = 64


def _layer(**modules):
    layer = nn.Module()
    for name, m in modules.items():
        layer.add_module(name, m)
    return layer


def _rms(eps=1e-6, width=D, dtype=torch.bfloat16):
    from transformers.models.qwen3.modeling_qwen3 import Qwen3RMSNorm

    norm = Qwen3RMSNorm(width, eps=eps)
    norm.weight.data.copy_(1 + 0.3 * torch.randn(width, generator=torch.Generator().manual_seed(1)))
    return norm.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e-3])
def test_norms_over_a_head_are_taken(dtype, eps):
    q, k = _rms(eps, dtype=dtype), _rms(eps, dtype=dtype)
    got = PagedAttentionLayer._head_norms(_layer(q_norm=q, k_norm=k), D)
    assert got[0] is q.weight and got[1] is k.weight and got[2] == eps
    assert PagedAttentionLayer._head_norms(_layer(k_norm=k), D) == (None, k.weight, eps)


def test_torch_norms_are_taken():
    q = nn.RMSNorm(D, eps=1e-5).to(torch.bfloat16)
    assert PagedAttentionLayer._head_norms(_layer(q_norm=q, k_norm=nn.Identity()), D) == (q.weight, None, 1e-5)
    q = nn.RMSNorm(D).to(torch.float16)  # eps None: that of its arithmetic
    assert PagedAttentionLayer._head_norms(_layer(q_norm=q), D)[2] == torch.finfo(torch.float32).eps


def test_no_norms():
    assert PagedAttentionLayer._head_norms(_layer(), D) == (None, None, 1e-6)


def _gemma():
    from transformers.models.gemma3.modeling_gemma3 import Gemma3RMSNorm

    return Gemma3RMSNorm(D).to(torch.bfloat16)


def _wrong_eps():
    norm = _rms(1e-3)
    norm.eps, norm.variance_epsilon = 1e-3, 1e-6
    norm.forward = lambda x: _rms(1e-3)(x)
    return norm


@pytest.mark.parametrize("modules", [
    lambda: dict(q_norm=nn.LayerNorm(D).to(torch.bfloat16)),
    lambda: dict(k_norm=nn.LayerNorm(D, bias=False)),
    lambda: dict(q_norm=_gemma()),
    lambda: dict(q_norm=_rms(width=8 * D), k_norm=_rms(width=2 * D)),
    lambda: dict(k_norm=nn.RMSNorm(D, elementwise_affine=False)),
    lambda: dict(q_norm=_rms(1e-3), k_norm=_rms(1e-6)),
    lambda: dict(q_norm=_wrong_eps()),
    lambda: dict(q_layernorm=_rms(), k_layernorm=_rms()),
    lambda: dict(q_norm=_rms(), k_norm=_rms(), attn_sub_norm=_rms()),
], ids=["layer norm", "layer norm without bias", "one plus weight", "all heads", "no weight",
        "two eps", "another eps", "other names", "a norm more"])
def test_other_norms_are_refused(modules):
    with pytest.raises(NotImplementedError):
        PagedAttentionLayer._head_norms(_layer(**modules()), D)
