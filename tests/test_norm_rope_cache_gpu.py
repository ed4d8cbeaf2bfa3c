"""Norms, rotation and cache write in one pass, and the 8-bit cache's read-back,
against their formulas in 64 bits.

Bounds (set before the first run).  With u the unit roundoff of the 16-bit type
(2^-8 bf16, 2^-11 fp16) and e = 2^-24:

* A sum of D <= 128 squares and what follows it (mean, 1 / sqrt at 2 ulp, two
  products) put a normalised y off by a relative 80 e < 2^-17; unnormalised it
  is exact.
* The reduced angle is rounded to fp32 (pi e) and the functions are within 2 ulp:
  cos and sin are off by 6 e.  A rotated value is off by (|y_lo| + |y_hi|) *
  (2^-17 + 8 e) at most, 2^-16 below.
* One rounding: u |z|, or half the smallest step of the type.
* A code is the value over its scale to nearest: the half step of
  ``_half_step`` with the fp32 error above, which moves the value by 2^-16 of
  |y_lo| + |y_hi| and the row's scale by the same share, and 2^-21 of the row's
  largest for the quantising arithmetic itself.

The read-back is code * scale rounded twice (to fp32, to 16 bits), the same
operations in torch: equal bit for bit.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
U = {dt: torch.finfo(dt).eps / 2 for dt in (torch.float16, torch.bfloat16)}
LEAST = {dt: torch.finfo(dt).smallest_normal * torch.finfo(dt).eps for dt in U}


def _inputs(rows, n_q, n_kv, D, dtype, seed, pad=0, blocks=None, far=False):
    """q, k, v as slices of one fused output (``pad`` spare columns), rows at random slots."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    qkv = torch.randn((rows, (n_q + 2 * n_kv) * D + pad), generator=g).to(dtype).cuda()
    blocks = blocks or (rows + 15) // 16 + 2
    slots = rng.permutation(blocks * 16)[:rows]
    pos = rng.integers(0, 2 ** 31 - 1 if far else 140000, rows)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    w = lambda: (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda()  # noqa: E731
    nq, nk = n_q * D, n_kv * D
    return dict(q=qkv[:, :nq].unflatten(1, (n_q, D)) if n_q else None,
                k=qkv[:, nq:nq + nk].unflatten(1, (n_kv, D)), v=qkv[:, nq + nk:nq + 2 * nk],
                positions=i32(pos), slot_mapping=i32(slots),
                inv_freq=(1.0 / (500000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))).cuda(),
                q_weight=w(), k_weight=w()), blocks


def _rotated(x, weight, pos, inv_freq, eps):
    """(z, |y_lo| + |y_hi| for each element) in 64 bits on the CPU."""
    y = x.double().cpu()
    if weight is not None:
        y = y * weight.double().cpu() / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    lo, hi = y.chunk(2, -1)
    size = (lo.abs() + hi.abs()).repeat(1, 1, 2)
    if inv_freq is None:
        return y, size
    a = (pos.double().cpu().unsqueeze(1) * inv_freq.double().cpu()).unsqueeze(1)
    cos, sin = torch.cos(a), torch.sin(a)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1), size


def _half_step(z, a, fmt):
    if fmt == INT8:
        return a / 254
    return torch.maximum(z.abs() * 2.0 ** -4, a / 448 * 2.0 ** -10)


def _near16(got, z, size, dtype):
    tol = U[dtype] * z.abs() + size * 2.0 ** -16 + LEAST[dtype]
    return float(((got.double().cpu() - z).abs() / tol).max())


def _near8(got, z, size, fmt):
    a = z.abs().amax(-1, keepdim=True)
    top = size.amax(-1, keepdim=True) * 2.0 ** -16
    tol = _half_step(z, a + top, fmt) + size * 2.0 ** -16 + top + a * 2.0 ** -21
    return float(((got.double().cpu() - z).abs() / tol).max())


def _slots_of(pool, slots):
    s = slots.long()
    return pool[s // 16, 0, s % 16], pool[s // 16, 1, s % 16]


CASES = [
    # rows, n_q, n_kv, D, dtype, spare columns
    (1, 32, 8, 128, torch.bfloat16, 0),
    (3, 4, 1, 64, torch.float16, 8),
    (70, 15, 5, 64, torch.bfloat16, 24),
    (33, 7, 7, 128, torch.float16, 0),
    (257, 64, 4, 64, torch.float16, 0),
    (19, 80, 16, 128, torch.bfloat16, 64),
    (5, 0, 3, 128, torch.float16, 0),
]


@pytest.mark.parametrize("norm", ["both", "k", "none"])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("fmt", [None, INT8, E4M3])
def test_against_the_formula(case, norm, fmt):
    rows, n_q, n_kv, D, dtype, pad = case
    a, blocks = _inputs(rows, n_q, n_kv, D, dtype, rows + D, pad)
    if norm != "both":
        a["q_weight"] = None
    if norm == "none":
        a["k_weight"] = None
    if fmt is None:
        cache = torch.full((blocks, 2, 16, n_kv, D), 7.0, dtype=dtype, device="cuda")
        before = cache.clone()
    else:
        cache = K.KVCache8.zeros(blocks, n_kv, D, fmt)
        cache.scales.fill_(3.0)
        cache.codes.view(torch.int8).fill_(1)
        before = cache.dequantize()
    kept = [t.clone() for t in (a["k"], a["v"])]
    got = K.norm_rope_and_cache(**a, cache=cache, eps=1e-5)
    assert torch.equal(a["k"], kept[0]) and torch.equal(a["v"], kept[1])
    args = (a["positions"], a["inv_freq"], 1e-5)
    if n_q:
        assert got.shape == (rows, n_q, D) and got.dtype == dtype
        assert _near16(got, *_rotated(a["q"], a["q_weight"], *args), dtype) <= 1
    else:
        assert got is None
    k, size = _rotated(a["k"], a["k_weight"], *args)
    v = a["v"].double().cpu().unflatten(1, (n_kv, D))
    pool = cache if fmt is None else cache.dequantize()
    kk, vv = _slots_of(pool, a["slot_mapping"])
    if fmt is None:
        assert _near16(kk, k, size, dtype) <= 1
        assert torch.equal(vv.cpu().double(), v)
    else:
        assert _near8(kk, k, size, fmt) <= 1
        assert _near8(vv, v, torch.zeros(()), fmt) <= 1
    # Every other slot is as it was.
    s = a["slot_mapping"].long()
    pool = pool.clone()
    pool[s // 16, :, s % 16] = before[s // 16, :, s % 16]
    assert torch.equal(pool, before)


@pytest.mark.parametrize("fmt", [None, E4M3])
def test_far_positions_and_in_place(fmt):
    """Positions up to 2^31: the angle's whole turns are taken off in 64 bits."""
    a, blocks = _inputs(40, 6, 2, 64, torch.float16, 5, pad=40, far=True)
    q = a["q"].clone()
    cache = torch.zeros((blocks, 2, 16, 2, 64), dtype=torch.float16, device="cuda") if fmt is None \
        else K.KVCache8.zeros(blocks, 2, 64, fmt)
    got = K.norm_rope_and_cache(**a, cache=cache, q_out=a["q"])
    assert got.data_ptr() == a["q"].data_ptr()
    z, size = _rotated(q, a["q_weight"], a["positions"], a["inv_freq"], 1e-6)
    assert _near16(got, z, size, torch.float16) <= 1


def test_same_rotation_as_the_unnormalised_write():
    """Without weights it is kernel 1's rotation, which rounds at each product."""
    a, blocks = _inputs(50, 8, 2, 128, torch.float16, 6)
    a["positions"] %= 2048
    a["q_weight"] = a["k_weight"] = None
    mine = torch.zeros((blocks, 2, 16, 2, 128), dtype=torch.float16, device="cuda")
    other = torch.zeros_like(mine)
    got = K.norm_rope_and_cache(**a, cache=mine)
    q = K.rope_reshape_and_cache(a["q"].contiguous(), a["k"], a["v"], a["positions"],
                                 a["slot_mapping"], a["inv_freq"], other)
    # Kernel 1 rounds cos, sin, both products and their sum (5 roundings of values up
    # to |y_lo| + |y_hi|) and the angle to fp32: 2048 * 2^-24.
    size = (a["q"].double().abs()[..., :64] + a["q"].double().abs()[..., 64:]).repeat(1, 1, 2)
    assert ((got.double() - q.double()).abs() <= size * (5 * 2.0 ** -11 + 2048 * 2.0 ** -24)).all()
    assert torch.equal(mine[:, 1], other[:, 1])


@pytest.mark.parametrize("fmt", [None, INT8])
def test_rows_that_cache_nothing(fmt):
    a, blocks = _inputs(6, 4, 2, 64, torch.bfloat16, 7)
    a["slot_mapping"][[1, 4]] = -1
    cache = torch.zeros((blocks, 2, 16, 2, 64), dtype=torch.bfloat16, device="cuda") if fmt is None \
        else K.KVCache8.zeros(blocks, 2, 64, fmt)
    got = K.norm_rope_and_cache(**a, cache=cache)
    z, size = _rotated(a["q"], a["q_weight"], a["positions"], a["inv_freq"], 1e-6)
    assert _near16(got, z, size, torch.bfloat16) <= 1
    pool = cache if fmt is None else cache.dequantize()
    assert int((pool != 0).flatten(3).any(3).all(1).sum()) == 4


def test_no_rows():
    a, blocks = _inputs(0, 4, 2, 64, torch.float16, 8, blocks=2)
    cache = K.KVCache8.zeros(2, 2, 64)
    assert K.norm_rope_and_cache(**a, cache=cache).shape == (0, 4, 64)


def test_bad_positions_and_slots_are_reported():
    a, blocks = _inputs(4, 4, 2, 64, torch.float16, 9)
    a["positions"][1] = -1
    a["slot_mapping"][2] = blocks * 16
    cache = K.KVCache8.zeros(blocks, 2, 64)
    K.norm_rope_and_cache(**a, cache=cache)
    assert K.error_word() == 16 | 1
    pool = cache.dequantize()
    assert int((pool != 0).flatten(3).any(3).all(1).sum()) == 2


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_values_that_are_no_numbers(fmt):
    """A head's row with an infinity or NaN reads as NaN; its neighbours are untouched."""
    a, blocks = _inputs(3, 4, 2, 128, torch.bfloat16, 10)
    a["k"][0, 1, 5], a["v"][1, 3], a["v"][1, 130] = float("nan"), float("inf"), -float("inf")
    a["v"][2, :128] = 0
    a["inv_freq"] = None
    a["k_weight"] = None
    cache = K.KVCache8.zeros(blocks, 2, 128, fmt)
    K.norm_rope_and_cache(**a, cache=cache)
    k, v = _slots_of(cache.dequantize(), a["slot_mapping"])
    assert torch.isnan(k[0, 1]).all() and torch.isnan(v[1]).all()
    assert torch.isfinite(k[0, 0]).all() and torch.isfinite(k[1:]).all() and torch.isfinite(v[[0, 2]]).all()
    assert (v[2, 0] == 0).all() and (v[2, 1] != 0).any()
    z = a["k"][1:].double().cpu()
    assert _near8(k[1:], z, torch.zeros(()), fmt) <= 1


def test_codes_are_those_of_the_torch_form():
    """Without norm and rotation both divide the same 16-bit values: equal codes but for
    values within 2^-21 of a tie, of which random ones have none in a few thousand."""
    a, blocks = _inputs(60, 2, 4, 64, torch.float16, 11)
    a["inv_freq"] = a["q_weight"] = a["k_weight"] = None
    for fmt in (INT8, E4M3):
        cache = K.KVCache8.zeros(blocks, 4, 64, fmt)
        K.norm_rope_and_cache(**a, cache=cache)
        s = a["slot_mapping"].long()
        codes, scales = K.quantize_cache8(a["k"], fmt)
        mine = cache.codes.view(torch.int8)[s // 16, 0, s % 16].view(fmt).float()
        apart = (mine - codes.float()).abs()
        assert (apart > 0).float().mean() < 1e-3
        assert torch.allclose(cache.scales[s // 16, :, 0, s % 16], scales, rtol=2.0 ** -23, atol=0)


# ── read-back ────────────────────────────────────────────────────────────────


def _cache(blocks, n_kv, D, fmt, seed):
    g = torch.Generator().manual_seed(seed)
    codes, scales = K.quantize_cache8(torch.randn((blocks, 2, 16, n_kv, D), generator=g), fmt)
    return K.KVCache8(codes.cuda(), scales.permute(0, 3, 1, 2).contiguous().cuda())


def _read_reference(cache, bt, lens, pool, dst):
    full = cache.dequantize().to(pool.dtype).cpu()
    want = pool.clone().cpu()
    for i, n in enumerate(lens):
        for j in range((n + 15) // 16):
            page = full[bt[i, j]].clone()
            page[:, max(0, n - 16 * j):] = 0
            want[dst[i, j]] = page
    return want


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("n_kv, D, lens", [
    (1, 64, [1]), (3, 64, [0, 15, 16, 17, 0, 100]), (8, 128, [33, 0, 129]), (5, 128, [16, 31]),
    (16, 64, list(range(40))), (2, 64, [3] * 300),
])
def test_read_back(n_kv, D, lens, fmt, dtype):
    rng = np.random.default_rng(D + n_kv)
    pages = [(n + 15) // 16 for n in lens]
    blocks, width = sum(pages) + 2, max(pages) + 2
    cache = _cache(blocks, n_kv, D, fmt, 1)
    # Unused entries of the tables are not looked at.
    bt, dst = np.full((len(lens), width), -7), np.full((len(lens), width), 1 << 30)
    order, to, at = rng.permutation(blocks), rng.permutation(blocks), 0
    for i, n in enumerate(pages):
        bt[i, :n], dst[i, :n] = order[at:at + n], to[at:at + n]
        at += n
    pool = torch.full((blocks, 2, 16, n_kv, D), 5.0, dtype=dtype, device="cuda")
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    want = _read_reference(cache, bt, lens, pool, dst)
    got = K.read_cache8(cache, i32(bt), i32(lens), pool, i32(dst))
    assert got is pool and torch.equal(pool.cpu(), want)


@pytest.mark.parametrize("n_kv, D, lens", [
    (64, 128, [20]), (33, 128, [5, 47]), (32, 128, [700, 0, 900]), (8, 128, [4095, 3]),
    (8, 128, [9000]), (5, 128, [1000]), (7, 64, [2000, 17]), (2, 128, [31, 1]),
])
def test_read_back_of_pages_shared_by_blocks(n_kv, D, lens):
    """Few pages, whose rows one, two, four or eight blocks share."""
    test_read_back(n_kv, D, lens, E4M3, torch.bfloat16)


@pytest.mark.parametrize("n_kv, D", [(2, 64), (8, 128)])
def test_read_back_into_a_pool_at_16_bytes(n_kv, D):
    """The pool starts between two 32-byte boundaries."""
    cache = _cache(4, n_kv, D, INT8, 4)
    size = 4 * 2 * 16 * n_kv * D
    memory = torch.full((size + 16,), 5.0, dtype=torch.float16, device="cuda")
    pool = memory[8:8 + size].view(4, 2, 16, n_kv, D)
    assert pool.data_ptr() % 32 == 16
    bt, dst, lens = np.array([[3, 0], [2, 0]]), np.array([[1, 3], [0, 2]]), [30, 16]
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    want = _read_reference(cache, bt, lens, pool, dst)
    assert torch.equal(K.read_cache8(cache, i32(bt), i32(lens), pool, i32(dst)).cpu(), want)
    assert (memory[:8] == 5).all() and (memory[8 + size:] == 5).all()


def test_wide_tables():
    """Tables far wider than the sequences, so many that a block takes several pages."""
    lens = [0] * 400
    lens[3], lens[200], lens[399] = 1000, 17, 16
    cache = _cache(70, 2, 64, INT8, 3)
    bt, dst = np.zeros((400, 130), np.int64), np.zeros((400, 130), np.int64)
    at = 0
    for i, n in enumerate(lens):
        for j in range((n + 15) // 16):
            bt[i, j], dst[i, j] = 69 - at, at
            at += 1
    pool = torch.full((70, 2, 16, 2, 64), 5.0, dtype=torch.float16, device="cuda")
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    want = _read_reference(cache, bt, lens, pool, dst)
    assert torch.equal(K.read_cache8(cache, i32(bt), i32(lens), pool, i32(dst)).cpu(), want)


def test_read_back_reports_bad_blocks():
    cache = _cache(3, 2, 64, INT8, 2)
    pool = torch.full((3, 2, 16, 2, 64), 5.0, dtype=torch.float16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bt, dst, lens = i32([[0, 3], [1, 2], [2, 0]]), i32([[0, 1], [-1, 2], [1, 0]]), i32([32, 32, 40])
    lens[2] = 0
    K.read_cache8(cache, bt, lens, pool, dst)
    assert K.error_word() == 2
    full = cache.dequantize().half()
    assert torch.equal(pool[0], full[0]) and torch.equal(pool[2], full[2]) and (pool[1] == 5).all()
    lens = i32([0, 0, 40])
    K.read_cache8(cache, bt, lens, pool, dst)  # three pages' worth, two in the table
    assert K.error_word() == 4
    assert torch.equal(pool[1], full[2]) and torch.equal(pool[0], full[0])


def test_calls_in_a_graph():
    """Write and read-back captured once, replayed on other inputs in the same memory."""
    a, blocks = _inputs(32, 4, 2, 64, torch.bfloat16, 12)
    a["slot_mapping"] = torch.arange(32, dtype=torch.int32, device="cuda")
    cache = K.KVCache8.zeros(blocks, 2, 64, E4M3)
    pool = torch.zeros((2, 2, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bt, lens = i32([[0, 1]]), i32([32])

    def both():
        q = K.norm_rope_and_cache(**a, cache=cache)
        K.read_cache8(cache, bt, lens, pool, bt)
        return q

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = both()
    a["q"].mul_(-0.5), a["k"].add_(0.25), a["v"].mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    got_q, got = q.clone(), pool.clone()
    want_q = both()
    assert torch.equal(got_q, want_q) and torch.equal(got, pool)
