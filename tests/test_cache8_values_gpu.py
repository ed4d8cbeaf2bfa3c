"""Decode attention over 8-bit caches whose values are out of the ordinary.

A stored value is code * scale whatever the scale's sign, and a token's V counts
by its weight: what it holds is of no account where its weight is nothing.

Bound of the built cases (set before the first run).  A score is off by at most
e_t = (D + 8) 2^-23 S_t, S_t the sum of its products' magnitudes times the scale,
and its weight by the same share, in the products with V and in the sum that they
are divided by; twice that is taken.  A weight times V's scale is rounded once to
fp16: 2^-11 of itself, or, where that is more, half of fp16's smallest step, 2^-25,
with the largest product of the warp's tokens at 2^10 or above: 2^-35 of the
largest, W = max_t p_t amax_t, for each of the n tokens (a code's 127 or 448 is
amax over its scale).  With A = sum_t p_t |V_t| and one rounding of the result (u):
    2 (sum_t p_t e_t |V_t| + |out| sum_t p_t e_t) + 2 * 2^-11 A + n 2^-35 W + u |out| + half of
the type's smallest step (fp16 2^-25, bf16 2^-134).

For fp16 outputs what the rounding to fp16 left is kept too (2^-22).  A weight's
logarithm is then the largest term: fp32 below 2^5 (2^-20, and 2^-22 of the exponential),
in cut sequences once more below 2^7 (2^-18), in the products and in the sum:
2^-16 A in place of 2 * 2^-11 A.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_cache8_decode_gpu import E4M3, INT8, U, _case, _reference, _worst
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


def _built(scores, sizes, G, D, dtype, fmt, seed):
    """One sequence, one kv head: K's element 0 gives token t about scores[t], V's largest
    magnitude is about sizes[t]."""
    n = len(scores)
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    pages = (n + 15) // 16
    order = rng.permutation(pages + 2)
    codes = torch.zeros((pages + 2, 2, 16, 1, D))
    scales = torch.zeros((pages + 2, 1, 2, 16))
    t = torch.arange(n)
    blk, slot = torch.from_numpy(order)[t // 16].long(), t % 16
    codes[blk, 0, slot, 0, 0] = 100.0
    scales[blk, 0, 0, slot] = torch.as_tensor(scores, dtype=torch.float32) * math.sqrt(D) / 8 / 100
    codes[blk, 1, slot, 0] = torch.randint(1, 5, (n, D), generator=g) * 32.0 - 1.0  # at most 127
    scales[blk, 0, 1, slot] = torch.as_tensor(sizes, dtype=torch.float32) / 128
    q = torch.zeros((1, G, D))
    q[..., 0] = 8.0
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(q=q.to(dtype).cuda(), cache=K.KVCache8(codes.to(fmt).cuda(), scales.cuda()),
                block_tables=i32(order[None, :pages]), seq_lens=i32([n]))


def _off(c, got, weights=2 * 2.0 ** -11, least=2.0 ** -35):
    """The largest error as a share of its bound."""
    q, cache, n = c["q"][0].double(), c["cache"], int(c["seq_lens"][0])
    G, D = q.shape
    ids = c["block_tables"][0].long()
    x = cache.codes.view(torch.int8)[ids].view(cache.codes.dtype).double()
    x = x * cache.scales[ids].double().permute(0, 2, 3, 1).unsqueeze(-1)
    k, v = (x[:, j, :, 0].flatten(0, 1)[:n] for j in (0, 1))
    p = torch.softmax(q @ k.T / math.sqrt(D), 1)
    e = (D + 8) * 2.0 ** -23 * (q.abs() @ k.abs().T) / math.sqrt(D)
    out, a = p @ v, p @ v.abs()
    w = (p * v.abs().amax(1)).amax(1, keepdim=True)
    tol = 2 * ((p * e) @ v.abs() + out.abs() * (p * e).sum(1, keepdim=True)) + weights * a \
        + n * least * w + U[got.dtype] * out.abs() \
        + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134)
    assert torch.isfinite(got).all()
    return float(((got[0].double() - out).abs() / tol).max())


@pytest.mark.parametrize("n, at", [(60, 3), (60, 59), (333, 200), (20000, 0), (20000, 11111)])
@pytest.mark.parametrize("up", [10, 30, 60, 100])
@pytest.mark.parametrize("G, D, dtype, fmt", [(4, 128, torch.bfloat16, INT8), (9, 64, torch.float16, E4M3),
                                              (16, 128, torch.float16, INT8)])
def test_a_token_without_weight_costs_the_others_nothing(G, D, dtype, fmt, up, at, n):
    """Its V is 2^up times the others', its weight 2^-220."""
    rng = np.random.default_rng(n + up)
    scores, sizes = rng.normal(size=n), np.exp2(rng.uniform(-1, 1, n))
    scores[at], sizes[at] = -150.0, 2.0 ** up
    c = _built(scores, sizes, G, D, dtype, fmt, n)
    assert _off(c, K.paged_decode_attention_cache8(**c)) <= 1


@pytest.mark.parametrize("n", [130, 3000])
@pytest.mark.parametrize("rise, fall", [(4, 6), (6, 4), (5, 5), (-4, -6), (-6, -4), (12, -3), (-12, 3)])
@pytest.mark.parametrize("G, D, dtype, fmt", [(4, 128, torch.bfloat16, E4M3), (12, 64, torch.bfloat16, INT8)])
def test_weights_and_values_that_drift_apart(G, D, dtype, fmt, rise, fall, n):
    """Weights rise by 2^rise a step (of 16 in all), V falls by 2^fall: the products' largest is where
    the weights' is, or at the other end, or everywhere."""
    step = np.arange(n) * 16 // n
    c = _built(math.log(2.0) * rise * step, np.exp2(-1.0 * fall * step), G, D, dtype, fmt, n)
    assert _off(c, K.paged_decode_attention_cache8(**c)) <= 1


@pytest.mark.parametrize("n", [5, 137, 2000, 30000])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("G, D", [(1, 64), (8, 64), (4, 128), (16, 64), (11, 128)])
def test_fp16_outputs_are_rounded_once(G, D, fmt, n):
    c = _case([n], G, 1, D, torch.float16, fmt, n + G, spare=False)
    assert _off(c, K.paged_decode_attention_cache8(**c), 2.0 ** -16) <= 1


@pytest.mark.parametrize("G, D, fmt", [(4, 128, INT8), (9, 64, E4M3)])
@pytest.mark.parametrize("size", [-99, -60, 60, 99])
def test_values_near_the_ends_of_fp32(size, G, D, fmt):
    """All of V tiny (products with weights of at most 2^104 leave fp16 2^-17 of the largest) or
    huge; most weights 2^-30 of the others."""
    rng = np.random.default_rng(3)
    n = 3000
    scores = np.where(rng.random(n) < 0.05, rng.normal(size=n), -30 * math.log(2.0))
    c = _built(scores, np.exp2(size + rng.uniform(0, 1, n)), G, D, torch.bfloat16, fmt, 4)
    got = K.paged_decode_attention_cache8(**c)
    assert _off(c, got, least=2.0 ** -17 if size == -99 else 2.0 ** -35) <= 1


def test_small_weights_beside_one_huge_value():
    """One token with half of the weight and V of 2^99; 20000 share the other half."""
    n = 20001
    scores, sizes = np.zeros(n), np.ones(n)
    scores[777], sizes[777] = math.log(n - 1.0), 2.0 ** 99
    c = _built(scores, sizes, 8, 64, torch.bfloat16, INT8, 5)
    assert _off(c, K.paged_decode_attention_cache8(**c)) <= 1
