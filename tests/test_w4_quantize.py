"""Rounding weights to 4-bit codes, whatever their size (no GPU).

A group's codes span its range in 15 steps (7 either way without zero points),
and a step is its scale.  Rounded to the type, a scale is off by a relative
roundoff, or by at most the type's smallest step where it is subnormal; a
weight is then within half a step of its code, half a step more where the zero
point's rounding moves a group's end past the last code, and 15 times what the
scale is off.
"""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200 import kernels as K


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("size", [4.0, 1e-1, 3e-3, 4e-4, 1e-4, 1e-5, 1e-6, 1e-7])
def test_codes_follow_the_weights_size(size, zero_points, dtype):
    g = torch.Generator().manual_seed(1)
    w = (torch.randn((16, 256), generator=g) * size).to(dtype)
    info = torch.finfo(dtype)
    least = info.smallest_normal * info.eps  # the type's smallest step
    for group in (32, 64, 128):
        q = K.quantize_w4(w, group, zero_points=zero_points)
        assert (q.scales > 0).all()
        parts = w.double().view(16, -1, group)
        if zero_points:
            step = (parts.amax(2).clamp(min=0) - parts.amin(2).clamp(max=0)) / 15
        else:
            step = parts.abs().amax(2) / 7
        off = torch.maximum(step * info.eps / 2, torch.full_like(step, least))
        bound = (1.0 if zero_points else 0.5) * (step + off) + 15 * off
        err = (q.dequantize().double() - w.double()).view(16, -1, group).abs().amax(2)
        assert (err <= bound).all(), float((err / bound).max())


def test_zero_groups_and_single_steps():
    w = torch.zeros((3, 64), dtype=torch.float16)
    w[1] = 2.0 ** -24          # the smallest fp16 number
    w[2, 5] = -2.0 ** -24
    for zero_points in (False, True):
        q = K.quantize_w4(w, 32, zero_points=zero_points)
        assert torch.equal(q.dequantize().half(), w)
