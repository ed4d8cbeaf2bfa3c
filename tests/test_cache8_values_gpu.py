"""Decode attention over 8-bit caches whose values are out of the ordinary.

A stored value is code * scale whatever the scale's sign, and a token's V counts
by its weight: what it holds is of no account where its weight is nothing.
"""

from __future__ import annotations

import pytest
import torch

from test_cache8_decode_gpu import E4M3, INT8, _case, _reference, _worst
from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("signs", ["all", "mixed"])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_of_either_sign(dtype, fmt, signs):
    """A cache of the caller's own may have negative scales, of K and of V."""
    c = _case([700, 1, 40, 16, 333], 32, 2, 128, dtype, fmt, 5)
    g = torch.Generator().manual_seed(6)
    scales = c["cache"].scales
    flip = torch.ones(scales.shape, dtype=torch.bool) if signs == "all" \
        else torch.rand(scales.shape, generator=g) < 0.5
    scales.mul_(torch.where(flip, -1.0, 1.0).cuda())
    assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1
