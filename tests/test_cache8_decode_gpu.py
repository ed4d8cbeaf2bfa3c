"""Decode attention over the 8-bit cache, against its formula in 64 bits.

Bound (set before the first run).  Codes are exact in 16 bits and so are
queries (bf16 ones scaled by a power of two; what that leaves below fp16's
range is 2^-24 of the row's largest), products are summed in fp32.  A score is
a sum of D products with an error of at most D * 2^-23 times the sum S of their
magnitudes; a weight times V's scale is rounded once to fp16 (2^-11) for the
product with V, its sum is not; the result is rounded once (u = 2^-8 bf16,
2^-11 fp16).  With A = sum_t p_t |V_t| an output is off by at most
    (2 * 2^-11 + 4 * (D + 8) * 2^-23 * scale * S) * A + u * |out| + least
(2 * 2^-11: the rounding, and the unrounded sum that it is divided by; D + 8:
scaling and the exponential's 2^-22), and least = 1e-6 of the largest |V|
covers results near zero and weights below fp16's range.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
U = {dt: torch.finfo(dt).eps / 2 for dt in (torch.float16, torch.bfloat16)}


def _case(lens, n_q, n_kv, D, dtype, fmt, seed, pad=0, spare=True, v_size=None, k_size=1.0, width=0):
    """Shuffled pages; every slot that no sequence owns holds codes and scales of no use
    (the largest code, scale NaN)."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    pages = [(n + 15) // 16 for n in lens]
    blocks = sum(pages) + 3
    order = rng.permutation(blocks)
    bt = np.zeros((len(lens), max([1, width] + pages)), np.int32)
    x = torch.randn((blocks, 2, 16, n_kv, D), generator=g)
    x[:, 0] *= k_size
    if v_size is not None:
        x[:, 1] *= torch.exp2(v_size * (2 * torch.rand((blocks, 16, n_kv, 1), generator=g) - 1))
    codes, scales = K.quantize_cache8(x, fmt)
    scales = scales.permute(0, 3, 1, 2).contiguous()
    owned = torch.zeros((blocks, 16), dtype=torch.bool)
    at = 0
    for i, n in enumerate(lens):
        bt[i, :pages[i]] = order[at:at + pages[i]]
        t = torch.arange(n)
        owned[torch.from_numpy(bt[i])[t // 16].long(), t % 16] = True
        at += pages[i]
    if spare:
        codes.view(torch.int8).masked_fill_(~owned[:, None, :, None, None], 127)
        scales.masked_fill_(~owned[:, None, None, :], float("nan"))
    q = torch.randn((len(lens), n_q * D + pad), generator=g).to(dtype).cuda()
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(q=q[:, :n_q * D].unflatten(1, (n_q, D)), cache=K.KVCache8(codes.cuda(), scales.cuda()),
                block_tables=i32(bt), seq_lens=i32(lens))


def _reference(c, scale=None):
    q, cache = c["q"].double(), c["cache"]
    B, n_q, D = q.shape
    n_kv = cache.codes.shape[3]
    G = n_q // n_kv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, big, mag = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    top = 0.0
    for i, n in enumerate(c["seq_lens"].tolist()):
        if n == 0:
            continue
        ids = c["block_tables"][i, : (n + 15) // 16].long()
        x = cache.codes.view(torch.int8)[ids].view(cache.codes.dtype).double()
        x = x * cache.scales[ids].double().permute(0, 2, 3, 1).unsqueeze(-1)
        k, v = (x[:, j].flatten(0, 1)[:n].repeat_interleave(G, 1) for j in (0, 1))
        p = torch.softmax(torch.einsum("hd,thd->ht", q[i], k) * scale, 1)
        out[i] = torch.einsum("ht,thd->hd", p, v)
        big[i] = torch.einsum("ht,thd->hd", p, v.abs())
        mag[i] = (torch.einsum("hd,thd->ht", q[i].abs(), k.abs()).amax(1) * scale)[:, None]
        top = max(top, float(v.abs().max()))
    return out, big, mag, top


def _worst(got, ref):
    out, big, mag, top = ref
    D = out.shape[2]
    tol = (2 * 2.0 ** -11 + 4 * (D + 8) * 2.0 ** -23 * mag) * big + U[got.dtype] * out.abs() + 1e-6 * top
    assert torch.isfinite(got).all()
    diff = (got.double() - out).abs()
    return float(torch.where(diff > 0, diff / tol, 0.0).max())


CASES = [
    # n_q, n_kv, D, dtype, fmt, lengths
    (32, 4, 64, torch.float16, INT8, [137]),
    (32, 8, 128, torch.bfloat16, E4M3, [1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 65]),
    (32, 8, 128, torch.bfloat16, INT8, [1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 65]),
    (1, 1, 64, torch.float16, E4M3, [300, 0, 1]),
    (16, 1, 128, torch.float16, INT8, [5000, 129, 7]),
    (16, 1, 64, torch.bfloat16, INT8, [1, 127, 128, 129, 2047]),
    (14, 2, 128, torch.bfloat16, INT8, [700, 33]),
    (6, 2, 64, torch.float16, E4M3, [513, 511, 3]),
    (9, 3, 128, torch.float16, INT8, [1000, 999]),
    (25, 5, 64, torch.bfloat16, E4M3, [400, 17]),
    (6, 6, 128, torch.bfloat16, INT8, [200, 16]),
    (28, 7, 64, torch.float16, INT8, [77, 401]),
    (36, 9, 128, torch.float16, E4M3, [150, 90]),
    (11, 11, 64, torch.bfloat16, INT8, [150, 90, 1100]),
    (52, 13, 128, torch.bfloat16, INT8, [150, 9]),
    (160, 16, 64, torch.float16, INT8, [260, 31]),
    (256, 16, 128, torch.bfloat16, E4M3, [260, 31]),
    (64, 64, 64, torch.float16, E4M3, [100, 5]),
    (32, 8, 128, torch.bfloat16, INT8, [20000]),
    (8, 2, 64, torch.float16, E4M3, [40001, 3, 0, 1]),
]


@pytest.mark.parametrize("case", CASES)
def test_against_the_formula(case):
    n_q, n_kv, D, dtype, fmt, lens = case
    c = _case(lens, n_q, n_kv, D, dtype, fmt, len(lens) + n_q)
    got = K.paged_decode_attention_cache8(**c)
    assert got.shape == c["q"].shape and got.dtype == dtype
    assert _worst(got, _reference(c)) <= 1
    assert (got[c["seq_lens"] == 0] == 0).all()


def _ragged(seed, n, most):
    return [int(x) for x in np.random.default_rng(seed).integers(0, most, n)]


@pytest.mark.parametrize("n, most, n_q, n_kv, D, dtype, fmt", [
    (64, 2048, 32, 4, 64, torch.float16, INT8),
    (33, 900, 16, 8, 128, torch.bfloat16, E4M3),
    (500, 40, 8, 2, 64, torch.bfloat16, INT8),
    (4096, 6, 4, 1, 64, torch.float16, INT8),
    (1500, 33, 8, 8, 128, torch.float16, E4M3),
    (300, 700, 16, 1, 128, torch.bfloat16, E4M3),
    # Tables of one to three pages: several heads a CTA.
    (4096, 16, 64, 4, 128, torch.bfloat16, INT8),
    (700, 17, 128, 8, 128, torch.float16, E4M3),
    (513, 32, 48, 16, 64, torch.bfloat16, INT8),
    (100, 33, 24, 12, 64, torch.float16, INT8),
    (100, 47, 21, 7, 64, torch.float16, E4M3),
])
def test_ragged_batches(n, most, n_q, n_kv, D, dtype, fmt):
    c = _case(_ragged(n, n, most), n_q, n_kv, D, dtype, fmt, n)
    assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1


def test_sequences_without_tokens():
    """No sequence has any: rows of zeros, whatever was there.  No sequences at all."""
    c = _case([0, 0, 0], 8, 2, 64, torch.float16, INT8, 2)
    out = torch.full((3, 8, 64), 9.0, dtype=torch.float16, device="cuda")
    assert (K.paged_decode_attention_cache8(**c, out=out) == 0).all()
    empty = dict(c, q=c["q"][:0], block_tables=c["block_tables"][:0], seq_lens=c["seq_lens"][:0])
    assert K.paged_decode_attention_cache8(**empty).shape == (0, 8, 64)


def test_strided_queries_given_scale_and_out():
    c = _case([90, 400, 0], 12, 4, 64, torch.bfloat16, INT8, 3, pad=72)
    assert not c["q"].is_contiguous()
    out = torch.full((3, 12, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    got = K.paged_decode_attention_cache8(**c, scale=0.31, out=out)
    assert got is out and _worst(got, _reference(c, 0.31)) <= 1
    flat = K.paged_decode_attention_cache8(c["q"].flatten(1).contiguous(), c["cache"],
                                           c["block_tables"], c["seq_lens"], 0.31)
    assert torch.equal(flat, got)


def test_runs_are_equal_bit_for_bit():
    c = _case([3000, 17, 800, 2999], 32, 8, 128, torch.bfloat16, INT8, 4)
    first = K.paged_decode_attention_cache8(**c)
    for _ in range(5):
        assert torch.equal(K.paged_decode_attention_cache8(**c), first)


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_of_very_different_size(fmt, dtype):
    """V's rows 2^-14 to 2^14 apart: the largest decide, and none leaves fp16's range."""
    c = _case([700, 40, 16], 8, 2, 128, dtype, fmt, 5, v_size=14.0)
    if dtype == torch.float16:
        c["cache"].scales[:, :, 1] *= 2.0 ** -4
    assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1


def test_sharp_and_flat_scores():
    """Scores hundreds apart (one token decides) and all equal."""
    for k_size in (60.0, 0.0):
        c = _case([1500, 64, 3], 16, 4, 64, torch.float16, INT8, 6, k_size=k_size)
        assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1


def test_many_small_weights_beside_a_large_one():
    """One token at weight 1/2, 30000 that share the other half: none of them is lost."""
    n, D = 30001, 64
    c = _case([n], 4, 1, D, torch.bfloat16, INT8, 7, k_size=0.0)
    q = torch.zeros((1, 4, D))
    q[..., 0] = 8.0
    c["q"] = q.to(torch.bfloat16).cuda()
    c["cache"].codes[:, 1] = 100  # V alike everywhere but at the one token
    c["cache"].scales[:, :, 1] = 0.01
    blk, slot = int(c["block_tables"][0, 700]), 5
    x = math.log(n - 1)  # its score above the others'
    c["cache"].codes[blk, 0, slot, 0, 0] = 127
    c["cache"].scales[blk, 0, 0, slot] = x / 127
    c["cache"].codes[blk, 1, slot] = -100
    ref = _reference(c)
    assert ref[0].abs().max() < 0.01 and _worst(K.paged_decode_attention_cache8(**c), ref) <= 1


def test_stored_rows_that_are_no_numbers():
    """NaN in a cached row reaches its own sequence and kv head alone; behind the length, nobody."""
    lens = [300, 40, 500]
    c = _case(lens, 8, 4, 64, torch.float16, INT8, 8)
    bt = c["block_tables"]
    c["cache"].scales[int(bt[0, 3]), 1, 0, 4] = float("nan")   # K of sequence 0, kv head 1
    c["cache"].scales[int(bt[2, 20]), 3, 1, 0] = float("nan")  # V of sequence 2, kv head 3
    got = K.paged_decode_attention_cache8(**c)
    bad = torch.isnan(got).all(2)
    want = torch.zeros_like(bad)
    want[0, 2:4] = True
    want[2, 6:8] = True
    assert torch.equal(bad, want) and torch.equal(torch.isnan(got).any(2), want)


def test_infinite_queries_give_nan():
    c = _case([50, 60], 4, 2, 64, torch.bfloat16, E4M3, 9)
    c["q"][0, 1, 7] = float("inf")
    got = K.paged_decode_attention_cache8(**c)
    assert torch.isnan(got[0, 1]).all()
    assert torch.isfinite(got[0, [0, 2, 3]]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4])
def test_queries_of_any_size(size):
    """bf16 queries are far outside fp16's range."""
    c = _case([200, 33], 8, 2, 128, torch.bfloat16, INT8, 10)
    q = c["q"].float() * size
    c["q"] = q.to(torch.bfloat16)
    c["cache"].scales[:, :, 0] *= 1.0 / size
    assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1


def test_bad_tables_are_reported():
    c = _case([40, 70], 8, 2, 64, torch.float16, INT8, 11)
    good = K.paged_decode_attention_cache8(**c)
    c["block_tables"][1, 2] = 10 ** 6
    got = K.paged_decode_attention_cache8(**c)
    assert K.error_word() == 2 and torch.equal(got[0], good[0])
    c = _case([40, 80], 8, 2, 64, torch.float16, INT8, 11)
    c["seq_lens"][1] = 81  # five pages in the table
    got = K.paged_decode_attention_cache8(**c)
    assert K.error_word() == 4
    c["seq_lens"][1] = 80
    assert _worst(got, _reference(c)) <= 1


def test_shared_pages():
    """Sequences with a common prefix read the same pages."""
    c = _case([330, 100, 340], 8, 2, 64, torch.bfloat16, INT8, 13)
    c["block_tables"][2, :20] = c["block_tables"][0, :20]
    assert _worst(K.paged_decode_attention_cache8(**c), _reference(c)) <= 1


def test_far_blocks():
    """Byte offsets past 2^31: blocks at both ends of a cache of more than 2 GiB."""
    n_kv, D = 16, 128
    blocks = (1 << 31) // (2 * 16 * n_kv * D) + 64
    small = _case([500, 30], 32, n_kv, D, torch.bfloat16, INT8, 12)
    codes = torch.zeros((blocks, 2, 16, n_kv, D), dtype=INT8, device="cuda")
    scales = torch.zeros((blocks, n_kv, 2, 16), device="cuda")
    n = small["cache"].codes.shape[0]
    codes[-n:], scales[-n:] = small["cache"].codes, small["cache"].scales
    big = dict(small, cache=K.KVCache8(codes, scales), block_tables=small["block_tables"] + (blocks - n))
    assert torch.equal(K.paged_decode_attention_cache8(**big), K.paged_decode_attention_cache8(**small))
    pool = torch.zeros((40, 2, 16, n_kv, D), dtype=torch.bfloat16, device="cuda")
    dst = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    K.read_cache8(big["cache"], big["block_tables"], big["seq_lens"], pool, dst)
    b = int(big["block_tables"][0, 1])
    want = (codes[b].float() * scales[b].permute(1, 2, 0).unsqueeze(-1)).to(torch.bfloat16)
    assert torch.equal(pool[1], want)


# ── workspaces, streams, graphs ──────────────────────────────────────────────


def test_one_workspace_for_every_shape():
    ws = K.DecodeWorkspace()
    for seed, (lens, n_q, n_kv, D) in enumerate([([3000, 5], 8, 2, 64), ([900] * 7, 32, 8, 128),
                                                 ([5000], 16, 1, 128), ([9] * 50, 8, 8, 64)]):
        c = _case(lens, n_q, n_kv, D, torch.float16, INT8, seed)
        got = K.paged_decode_attention_cache8(**c, workspace=ws)
        assert torch.equal(got, K.paged_decode_attention_cache8(**c))
    buf = next(iter(ws._buf.values()))
    assert not buf[: 1 << 20].any()
    # The 16-bit call takes the same one.
    pool = torch.randn((60, 2, 16, 2, 64), dtype=torch.float16, device="cuda")
    q = torch.randn((1, 8, 64), dtype=torch.float16, device="cuda")
    bt = torch.arange(60, dtype=torch.int32, device="cuda").view(1, 60)
    n = torch.tensor([950], dtype=torch.int32, device="cuda")
    assert torch.equal(K.paged_decode_attention(q, pool, bt, n, workspace=ws),
                       K.paged_decode_attention(q, pool, bt, n))


def test_workspaces_that_are_refused():
    c = _case([100], 8, 2, 64, torch.float16, INT8, 1)
    with pytest.raises(RuntimeError):
        K.paged_decode_attention_cache8(**c, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    big = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        K.paged_decode_attention_cache8(**c, workspace=big[16:])
    with pytest.raises(NotImplementedError):
        K.paged_decode_attention_cache8(**_case([10], 17, 1, 64, torch.float16, INT8, 1))


def test_two_streams_at_once():
    cases = [_case([4000, 900], 32, 8, 128, torch.bfloat16, INT8, s) for s in (1, 2)]
    want = [K.paged_decode_attention_cache8(**c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for j, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[j].append(K.paged_decode_attention_cache8(**c))
    torch.cuda.synchronize()
    for j in (0, 1):
        assert all(torch.equal(g, want[j]) for g in got[j])


def test_two_graphs_replayed_at_once():
    """Graphs captured without a workspace have their own: replays may overlap."""
    cases = [_case([4000, 900, 0, 17], 32, 4, 64, torch.float16, E4M3, s) for s in (3, 4)]
    want = [K.paged_decode_attention_cache8(**c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.paged_decode_attention_cache8(**c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    # Other lengths in the same memory.
    cases[0]["seq_lens"].copy_(torch.tensor([3999, 1, 16, 0], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    cases[0]["cache"].scales.nan_to_num_(nan=1.0)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert _worst(outs[0], _reference(cases[0])) <= 1


def test_write_then_attend_in_one_stream():
    """Prompt, then decode steps: each attends to what the writes before it stored."""
    g = torch.Generator().manual_seed(20)
    n_q, n_kv, D, dtype = 8, 2, 64, torch.bfloat16
    cache = K.KVCache8.zeros(12, n_kv, D, INT8)
    bt = torch.tensor([[4, 9, 1, 7]], dtype=torch.int32, device="cuda")
    inv = (1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))).cuda()
    w = torch.ones(D, dtype=dtype, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    n = 30
    qkv = torch.randn((n + 6, (n_q + 2 * n_kv) * D), generator=g).to(dtype).cuda()
    for at in [list(range(n))] + [[n + i] for i in range(6)]:
        rows = qkv[at]
        slots = [int(bt[0, t // 16]) * 16 + t % 16 for t in at]
        q = K.norm_rope_and_cache(rows[:, :n_q * D], rows[:, n_q * D:(n_q + n_kv) * D],
                                  rows[:, (n_q + n_kv) * D:], i32(at), i32(slots), inv, cache, w, w)
        lens = i32([at[-1] + 1])
        got = K.paged_decode_attention_cache8(q[-1:], cache, bt, lens)
        c = dict(q=q[-1:], cache=cache, block_tables=bt, seq_lens=lens)
        assert _worst(got, _reference(c)) <= 1
