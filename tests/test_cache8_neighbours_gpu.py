"""Outputs beside their inputs in one buffer."""

from __future__ import annotations

import pytest
import torch

from test_cache8_decode_gpu import INT8, _case
from test_norm_rope_cache_gpu import _inputs
from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_rotated_queries_behind_the_values(rows):
    n_q, n_kv, D = 6, 2, 64
    a, blocks = _inputs(rows, n_q, n_kv, D, torch.bfloat16, 3, pad=n_q * D)
    whole = a["q"].as_strided((rows, (2 * n_q + 2 * n_kv) * D), (a["q"].stride(0), 1))
    want = K.norm_rope_and_cache(**a, cache=K.KVCache8.zeros(blocks, n_kv, D))
    kept = whole[:, :(n_q + 2 * n_kv) * D].clone()
    out = whole[:, (n_q + 2 * n_kv) * D:]
    got = K.norm_rope_and_cache(**a, cache=K.KVCache8.zeros(blocks, n_kv, D), q_out=out)
    assert got is out and torch.equal(out.unflatten(1, (n_q, D)), want)
    assert torch.equal(whole[:, :(n_q + 2 * n_kv) * D], kept)


def test_outputs_in_the_place_of_keys_are_refused():
    a, blocks = _inputs(5, 4, 4, 64, torch.float16, 4)
    with pytest.raises(ValueError, match="overlaps"):
        K.norm_rope_and_cache(**a, cache=K.KVCache8.zeros(blocks, 4, 64), q_out=a["k"])


def test_attention_beside_and_over_its_queries():
    c = _case([300, 40], 8, 2, 64, torch.float16, INT8, 1)
    want = K.paged_decode_attention_cache8(**c)
    both = torch.empty((4, 8, 64), dtype=torch.float16, device="cuda")
    both[:2] = c["q"]
    q, out = both[:2], both[2:]
    assert torch.equal(K.paged_decode_attention_cache8(**{**c, "q": q}, out=out), want)
    with pytest.raises(ValueError, match="overlaps"):
        K.paged_decode_attention_cache8(**{**c, "q": q}, out=both[1:3])
