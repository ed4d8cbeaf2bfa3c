"""Joins of cut sequences in decode attention over the 8-bit cache.

A long sequence is cut between most of the GPU's CTAs; the last to arrive reads
what the others have published, in two rounds where there are many.  Whoever
that is, the result is the same bit for bit, call after call, and the counters
are left at zero.  A record that is read before it is there shows as another
result: the workspace holds an earlier call's records of other values.
"""

from __future__ import annotations

import pytest
import torch

from test_cache8_decode_gpu import E4M3, INT8, _case, _reference, _worst
from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu

CASES = [
    # n_q, n_kv, D, dtype, fmt, lengths: one run of pieces over all CTAs, several, runs that
    # start and end inside a CTA
    (16, 1, 128, torch.bfloat16, INT8, [40000]),
    (4, 1, 64, torch.float16, E4M3, [70001]),
    (32, 8, 128, torch.bfloat16, E4M3, [9001, 4000, 12345]),
    (8, 2, 64, torch.float16, INT8, [5000, 2999, 17, 5003, 4001, 16]),
    (10, 5, 128, torch.float16, INT8, [3001, 7, 6500]),
]


@pytest.mark.parametrize("case", CASES)
def test_joins_after_other_calls(case):
    n_q, n_kv, D, dtype, fmt, lens = case
    a, b = (_case(lens, n_q, n_kv, D, dtype, fmt, seed) for seed in (1, 2))
    ws = K.DecodeWorkspace()
    want = [K.paged_decode_attention_cache8(**c) for c in (a, b)]
    for c, w in zip((a, b), want):
        assert _worst(w, _reference(c)) <= 1
    for _ in range(40):
        for c, w in zip((a, b), want):
            assert torch.equal(K.paged_decode_attention_cache8(**c, workspace=ws), w)
    buf = next(iter(ws._buf.values()))
    assert not buf[: 1 << 20].any()
