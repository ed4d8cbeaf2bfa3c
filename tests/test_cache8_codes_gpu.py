"""Codes of 16-bit values: the ones that the exact quotient is nearest to, ties to even.

16-bit values times 127 or 448 are exact in 64 bits, and so is their quotient by the
row's largest where it lies on a tie; where it does not, it is at least 2^-21 of
itself away from one (a ratio of whole numbers of 11 bits and 9), so that 64
bits decide as the exact quotient does.  Every code is equal, therefore.
"""

from __future__ import annotations

import pytest
import torch

from vllm_mps_b200 import kernels as K

INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _rows(n, d, dtype, size, seed):
    """Random rows; some values are halves, quarters, 3/16 and 17/32 of their row's largest, where ties are."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, d), generator=g)
    a = x.abs().amax(1, keepdim=True).to(dtype).float()
    share = torch.tensor([0.5, -0.5, 0.25, 3 / 16, -17 / 32, 3 / 254, -5 / 254, 99 / 254])
    x[:, :8] = torch.where(x[:, :8].abs() < a, a * share, x[:, :8])
    return (x * size).to(dtype)


def _nearest(x, fmt):
    """Values of the codes of rows ``x``, in 64 bits."""
    top = K._CACHE_TOP[fmt]
    y = x.double() * top / x.double().abs().amax(-1, keepdim=True)
    if fmt == INT8:
        return torch.round(y)
    # e4m3: four significant bits, exponents from -6 up.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


CASES = [(torch.float16, 1.0), (torch.float16, 2.0 ** -8), (torch.float16, 2.0 ** 12),
         (torch.bfloat16, 1.0), (torch.bfloat16, 2.0 ** -90), (torch.bfloat16, 2.0 ** 125)]


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dtype, size", CASES)
def test_torch_form(dtype, size, fmt):
    x = _rows(2000, 64, dtype, size, 1)
    codes, scales = K.quantize_cache8(x, fmt)
    assert torch.equal(codes.double(), _nearest(x, fmt))
    assert torch.equal(scales, x.float().abs().amax(1) / K._CACHE_TOP[fmt])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dtype, size", CASES)
def test_written_codes(dtype, size, fmt, D):
    n_kv, rows = 4, 1000
    k, v = (_rows(rows * n_kv, D, dtype, size, seed).view(rows, n_kv, D) for seed in (1, 2))
    cache = K.KVCache8.zeros((rows + 15) // 16, n_kv, D, fmt)
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    assert K.norm_rope_and_cache(None, k.cuda(), v.cuda(), None, slots.cuda(), None, cache) is None
    s = slots.long().cuda()
    codes = cache.codes.view(torch.int8)
    for kind, x in ((0, k), (1, v)):
        got = codes[s // 16, kind, s % 16].view(fmt).double().cpu()
        assert torch.equal(got, _nearest(x, fmt))
        assert torch.equal(cache.scales[s // 16, :, kind, s % 16].cpu(),
                           x.float().abs().amax(-1) / K._CACHE_TOP[fmt])
