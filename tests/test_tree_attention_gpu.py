"""Attention of drafted tokens over the paged cache, against its formula in 64 bits.

Bound (set before the first run).  The kernel multiplies exact 16-bit
operands with fp32 accumulation, rounds the softmax weights once to the
16-bit type (unit roundoff u = 2^-8 bf16, 2^-11 fp16) for the product with V,
and rounds the result once.  A score is a sum of D products with an fp32
error of at most D * 2^-23 times the sum of their magnitudes S, so a weight
is off by a relative 2 * D * 2^-23 * scale * S at most (its own score and the
normalisation); with A = sum_t p_t |V_t| an output is off by at most
    (2u + 4 * D * 2^-23 * scale * S) * A + u * |out|
(2u: the rounding of a weight, and the same again in the unrounded sum it is
divided by, plus the approximate exponential's 2^-22), and 1e-6 covers
results near zero.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from vllm_mps_b200.core.draft_tree import DraftTree

pytestmark = pytest.mark.gpu

U = {dt: torch.finfo(dt).eps / 2 for dt in (torch.float16, torch.bfloat16)}  # unit roundoff


def _random_tree(rng, n):
    return DraftTree([-1] + [int(rng.integers(max(0, (i - 1) // 3), i)) for i in range(1, n)])


def _case(dev, seqs, n_q, n_kv, D, dtype, seed, q_pad=0, words=None, spare=float("nan"), q_scale=1.0):
    """``seqs``: (ctx, nodes, query rows = the last of the nodes).  Every slot that no
    sequence owns holds ``spare``."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    lens = [c + n for c, n, _ in seqs]
    pages = [(x + 15) // 16 for x in lens]
    order = rng.permutation(sum(pages) + 3)
    bt = np.zeros((len(seqs), max(1, max(pages))), np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = order[at:at + n]
        at += n
    pool = torch.full((len(order), 2, 16, n_kv, D), spare, dtype=torch.float32)
    for i, n in enumerate(lens):
        kv = torch.randn((n, 2, n_kv, D), generator=g)
        t = torch.arange(n)
        pool[torch.from_numpy(bt[i])[t // 16].long(), :, t % 16] = kv
    trees = [_random_tree(rng, n) if n else None for _, n, _ in seqs]
    words = words or max(1, max((n + 31) // 32 for _, n, _ in seqs))
    rows = [t.mask(words)[n - r:] for t, (_, n, r) in zip(trees, seqs) if r]
    total = sum(r for _, _, r in seqs)
    mask = np.concatenate(rows) if rows else np.zeros((0, words), np.int32)
    q = torch.randn((total, n_q * D + q_pad), generator=g) * q_scale
    cu = np.cumsum([0] + [r for _, _, r in seqs])[:-1]
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    qd = q.to(dtype).to(dev)
    return dict(q=qd[:, :n_q * D].unflatten(1, (n_q, D)), pool=pool.to(dtype).to(dev),
                bt=i32(bt), ctx=i32([c for c, _, _ in seqs]), lens=i32(lens),
                q_lens=i32([r for _, _, r in seqs]), cu=i32(cu),
                mask=i32(mask).view(total, words), max_q=max(r for _, _, r in seqs), seqs=seqs)


def _call(K, c, **kw):
    return K.paged_tree_attention(c["q"], c["pool"], c["bt"], c["ctx"], c["lens"], c["q_lens"],
                                  c["cu"], c["mask"], c["max_q"], **kw)


def _reference(c, scale=None, mask=None):
    """(out, A, scale * S) per element in 64 bits, on the CPU, one row at a time."""
    q, pool = c["q"].double().cpu(), c["pool"].double().cpu()
    mask = (c["mask"] if mask is None else mask).cpu().numpy().view(np.uint32)
    n_q, D = q.shape[1:]
    n_kv = pool.shape[3]
    G = n_q // n_kv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, big, mag = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    bt, at = c["bt"].cpu(), 0
    for i, (ctx, n, r) in enumerate(c["seqs"]):
        ids = bt[i, : (ctx + n + 15) // 16].long()
        k = pool[ids, 0].flatten(0, 1)[: ctx + n]
        v = pool[ids, 1].flatten(0, 1)[: ctx + n]
        for row in range(at, at + r):
            see = [t < ctx or (t - ctx < 32 * mask.shape[1]
                               and bool((mask[row, (t - ctx) // 32] >> ((t - ctx) % 32)) & 1))
                   for t in range(ctx + n)]
            see = torch.tensor(see, dtype=torch.bool)
            if not see.any():
                continue
            kk, vv = k[see].repeat_interleave(G, 1), v[see].repeat_interleave(G, 1)
            s = torch.einsum("hd,thd->ht", q[row], kk) * scale
            p = torch.softmax(s, 1)
            out[row] = torch.einsum("ht,thd->hd", p, vv)
            big[row] = torch.einsum("ht,thd->hd", p, vv.abs())
            mag[row] = (torch.einsum("hd,thd->ht", q[row].abs(), kk.abs()).amax(1) * scale)[:, None]
        at += r
    return out, big, mag


def _check(got, ref, dtype, D):
    out, big, mag = ref
    u = U[dtype]
    tol = (2 * u + 4 * D * 2.0 ** -23 * mag) * big + u * out.abs() + 1e-6
    diff = (got.double().cpu() - out).abs()
    assert torch.isfinite(got).all()
    worst = (diff / tol).max().item() if diff.numel() else 0.0
    assert worst <= 1.0, worst


CASES = [
    # n_q, n_kv, D, dtype, [(ctx, nodes, query rows)]
    (32, 4, 64, torch.float16, [(137, 8, 8)]),
    (8, 2, 128, torch.bfloat16, [(0, 1, 1), (1, 1, 1), (15, 1, 1), (16, 1, 1), (300, 1, 1)]),
    # Nothing cached, trees that end inside and at the edges of pages and key tiles.
    (8, 2, 64, torch.float16, [(0, 5, 5), (0, 64, 64), (0, 65, 65), (63, 1, 1), (64, 2, 2)]),
    # Ragged contexts and trees, a sequence without rows between others.
    (32, 8, 128, torch.bfloat16, [(1000, 26, 26), (3, 7, 7), (200, 0, 0), (129, 33, 33)]),
    # Query rows that are only the last level of a tree.
    (16, 8, 128, torch.float16, [(250, 17, 4), (77, 21, 3)]),
    # Every ratio of query to kv heads, powers of two or not.
    (4, 4, 64, torch.bfloat16, [(70, 40, 40)]),
    (9, 3, 128, torch.float16, [(90, 13, 13), (10, 50, 50)]),
    (10, 2, 64, torch.float16, [(90, 13, 13), (10, 30, 30)]),
    (7, 1, 128, torch.bfloat16, [(130, 20, 20), (1, 1, 1)]),
    (32, 2, 128, torch.float16, [(333, 20, 20), (0, 9, 9)]),
    (26, 2, 64, torch.bfloat16, [(40, 11, 11)]),
    # More than one row tile (rows x heads above 128, above 256), many kv heads.
    (64, 8, 128, torch.bfloat16, [(515, 64, 64), (80, 40, 40)]),
    (16, 1, 64, torch.float16, [(100, 64, 64), (100, 3, 3)]),
    # Long enough to be cut into pieces, next to short ones.
    (8, 2, 128, torch.float16, [(9000, 6, 6), (40, 6, 6), (0, 2, 2)]),
    (4, 1, 64, torch.bfloat16, [(20011, 3, 3)]),
    # Trees above one and two mask words.
    (4, 2, 64, torch.float16, [(33, 100, 100), (8, 130, 2)]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_formula(cuda_device, case):
    from vllm_mps_b200 import kernels as K

    n_q, n_kv, D, dtype, seqs = CASES[case]
    c = _case(cuda_device, seqs, n_q, n_kv, D, dtype, seed=case)
    got = _call(K, c)
    torch.cuda.synchronize()
    assert K.error_word(cuda_device) == 0
    _check(got, _reference(c), dtype, D)
    again = _call(K, c)
    assert torch.equal(got, again)  # the order of sums is fixed


def test_many_short_sequences(cuda_device):
    from vllm_mps_b200 import kernels as K

    rng = np.random.default_rng(3)
    seqs = []
    for _ in range(300):
        n = int(rng.integers(1, 6))
        seqs.append((int(rng.integers(0, 70)), n, n))
    c = _case(cuda_device, seqs, 4, 2, 64, torch.float16, seed=1)
    _check(_call(K, c), _reference(c), torch.float16, 64)


@pytest.mark.parametrize("ctx,n_kv,D", [(3000, 1, 128), (60000, 1, 64), (33000, 2, 128)])
def test_sequences_in_many_pieces(cuda_device, ctx, n_kv, D):
    """One sequence over the whole machine: its pieces are joined in groups, those again."""
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(ctx, 5, 5)], 3 * n_kv, n_kv, D, torch.float16, seed=ctx)
    got = _call(K, c)
    _check(got, _reference(c), torch.float16, D)
    for _ in range(5):
        assert torch.equal(got, _call(K, c))  # whichever piece comes last


def test_large_scores_and_scale(cuda_device):
    """Scores far apart (one key takes all) and a scale of the caller's."""
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(700, 20, 20), (5, 3, 3)], 8, 2, 128, torch.bfloat16, seed=5, q_scale=12.0)
    _check(_call(K, c, scale=0.7), _reference(c, scale=0.7), torch.bfloat16, 128)
    # Scores that grow along the sequence: the running maximum is raised many times.
    n = 1300
    c = _case(cuda_device, [(n, 4, 4)], 4, 2, 64, torch.float16, seed=6)
    ramp = torch.linspace(0.01, 8.0, n + 4, device=cuda_device)
    t = torch.arange(n + 4, device=cuda_device)
    blk = c["bt"][0, (t // 16)].long()
    c["q"][:] = 1.0
    c["pool"][blk, 0, t % 16] = ramp.half()[:, None, None].expand(-1, 2, 64)
    _check(_call(K, c, scale=0.25), _reference(c, scale=0.25), torch.float16, 64)


def test_strided_queries_out_and_workspace(cuda_device):
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    c = _case(dev, [(100, 12, 12), (31, 5, 5)], 8, 2, 128, torch.float16, seed=8, q_pad=2 * 2 * 128)
    assert not c["q"].is_contiguous()
    ref = _reference(c)
    got = _call(K, c)
    _check(got, ref, torch.float16, 128)
    need = K.paged_tree_attention_workspace_bytes(2, c["max_q"], 8, 2, 128, torch.float16)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)  # NaN patterns: never read back
    buf = torch.full((18, 8, 128), 7.0, dtype=torch.float16, device=dev)
    out = _call(K, c, out=buf[:17], workspace=ws)
    assert out.data_ptr() == buf.data_ptr()
    assert torch.equal(out, got)
    assert (buf[17] == 7.0).all()  # nothing past the rows is written


def test_rows_that_see_nothing_are_zero(cuda_device):
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(0, 6, 6), (20, 4, 4), (0, 70, 70)], 8, 2, 64, torch.bfloat16, seed=9)
    c["mask"][2] = 0          # no context and no draft: an empty row
    c["mask"][7] = 0          # the context alone
    c["mask"][10 + 30] = 0
    got = _call(K, c)
    _check(got, _reference(c), torch.bfloat16, 64)
    assert (got[2] == 0).all() and (got[10 + 30] == 0).all()


def test_masks_that_are_no_tree(cuda_device):
    """Any bits: a draft may see later drafts, or not itself; bits past the end are ignored."""
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(50, 40, 40), (3, 9, 9)], 4, 2, 128, torch.float16, seed=10, words=3)
    g = torch.Generator().manual_seed(2)
    c["mask"].copy_(torch.randint(-2 ** 31, 2 ** 31, c["mask"].shape, generator=g).to(torch.int32))
    _check(_call(K, c), _reference(c), torch.float16, 128)


def test_drafts_past_the_mask_are_not_seen(cuda_device):
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(10, 50, 5)], 4, 2, 64, torch.float16, seed=11)
    c["mask"] = c["mask"][:, :1].contiguous()
    _check(_call(K, c), _reference(c), torch.float16, 64)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_unseen_slots_take_no_part(cuda_device, bad):
    """Stale slots and drafts outside a row's mask may hold anything; rows that do see
    such a draft carry it."""
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    for ctx, n in ((60, 30), (5, 64), (130, 3)):
        c = _case(dev, [(ctx, n, n), (40, 4, 4)], 8, 2, 128, torch.float16, seed=12, spare=bad)
        node = n // 2
        clean = _case(dev, [(ctx, n, n), (40, 4, 4)], 8, 2, 128, torch.float16, seed=12, spare=0.0)
        ref = _reference(clean)
        t = ctx + node
        blk = int(c["bt"][0, t // 16])
        sees = (c["mask"][:n, node // 32].cpu() >> (node % 32)) & 1
        sees = torch.cat([sees.bool(), torch.zeros(4, dtype=torch.bool)])
        for part in (0, 1):
            pool = c["pool"].clone()
            pool[blk, part, t % 16, :, 5] = bad
            got = _call(K, dict(c, pool=pool))
            torch.cuda.synchronize()
            blind = ~sees
            _check(got[blind.to(dev)], tuple(x[blind] for x in ref), torch.float16, 128)
            seeing = got[sees.to(dev)]
            if part == 1:  # a bad value column reaches exactly that column
                if math.isnan(bad):
                    assert torch.isnan(seeing[..., 5]).all()
                else:
                    assert (seeing[..., 5] == bad).all()
                others = torch.cat([seeing[..., :5], seeing[..., 6:]], -1)
                assert torch.isfinite(others).all()
            elif math.isnan(bad):
                assert torch.isnan(seeing).all()


def test_same_as_decode_and_prefill(cuda_device):
    """One row a sequence is a decode step; a chain of drafts is a causal chunk."""
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    ctx = [0, 17, 300, 1029]
    c = _case(dev, [(x, 1, 1) for x in ctx], 32, 4, 64, torch.float16, seed=13, spare=0.0)
    dec = K.paged_decode_attention(c["q"].contiguous(), c["pool"], c["bt"], c["lens"])
    torch.testing.assert_close(_call(K, c).float(), dec.float(), atol=2e-3, rtol=2e-3)
    c = _case(dev, [(x, 20, 20) for x in ctx], 32, 8, 128, torch.float16, seed=14, spare=0.0)
    chain = DraftTree([-1] + list(range(19))).mask()
    c["mask"].copy_(torch.from_numpy(np.tile(chain, (4, 1))))
    pre = K.paged_prefill_attention(c["q"], c["pool"], c["bt"], c["ctx"], c["q_lens"], c["cu"], 20)
    torch.testing.assert_close(_call(K, c).float(), pre.float(), atol=2e-3, rtol=2e-3)


def test_other_streams_and_graphs(cuda_device):
    """Calls on two streams at once, and a captured call replayed on new inputs."""
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    a = _case(dev, [(5000, 16, 16)], 16, 4, 128, torch.float16, seed=15)
    b = _case(dev, [(4000, 9, 9)], 16, 4, 128, torch.float16, seed=16)
    want_a, want_b = _call(K, a), _call(K, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    outs = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            outs.append((_call(K, a), want_a))
        with torch.cuda.stream(s2):
            outs.append((_call(K, b), want_b))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _call(K, a)
    a["q"].copy_(a["q"].flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, _call(K, a))


def test_empty_calls(cuda_device):
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(20, 0, 0), (3, 0, 0)], 8, 2, 64, torch.float16, seed=17)
    assert _call(K, c).shape == (0, 8, 64)
    none = dict(c, bt=c["bt"][:0], ctx=c["ctx"][:0], lens=c["lens"][:0], q_lens=c["q_lens"][:0],
                cu=c["cu"][:0])
    assert _call(K, none).shape == (0, 8, 64)


def test_bad_indices_are_reported_and_skipped(cuda_device):
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    c = _case(dev, [(100, 5, 5), (50, 3, 3), (70, 2, 2)], 8, 2, 64, torch.float16, seed=18)
    want = _call(K, c)
    bt = c["bt"].clone()
    bt[1, 1] = c["pool"].shape[0] + 5
    got = _call(K, dict(c, bt=bt))
    assert K.error_word(dev) & 2
    assert torch.equal(got[:5], want[:5]) and torch.equal(got[8:], want[8:])
    lens = c["lens"].clone()
    lens[0] = 16 * c["bt"].shape[1] + 1  # one slot more than the table holds
    got = _call(K, dict(c, lens=lens))
    assert K.error_word(dev) & 4
    assert torch.equal(got[5:], want[5:])
    cu = c["cu"].clone()
    cu[2] = 9  # rows 9, 10 of 10
    out = torch.zeros_like(want)
    got = _call(K, dict(c, cu=cu), out=out)
    assert K.error_word(dev) & 64
    assert torch.equal(got[:8], want[:8])
    got = K.paged_tree_attention(c["q"], c["pool"], c["bt"], c["ctx"], c["lens"], c["q_lens"],
                                 c["cu"], c["mask"], 3)  # the first sequence has 5 rows
    assert K.error_word(dev) & 64
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[5:], want[5:])


def test_refusals(cuda_device):
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    c = _case(dev, [(20, 4, 4)], 8, 2, 64, torch.float16, seed=19)
    with pytest.raises(TypeError):
        _call(K, dict(c, q=c["q"].bfloat16()))
    with pytest.raises(TypeError):
        _call(K, dict(c, mask=c["mask"].long()))
    with pytest.raises(ValueError):
        _call(K, dict(c, mask=c["mask"][:2]))
    with pytest.raises(ValueError):
        _call(K, dict(c, ctx=c["ctx"][:0]))
    with pytest.raises(ValueError):
        _call(K, dict(c, q=c["q"].transpose(0, 1).contiguous().transpose(0, 1)))
    with pytest.raises(ValueError):
        _call(K, c, scale=float("nan"))
    with pytest.raises(RuntimeError, match="workspace"):
        _call(K, c, workspace=torch.empty(8, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError, match="CUDA"):
        _call(K, dict(c, ctx=c["ctx"].cpu()))
    with pytest.raises(NotImplementedError):
        _call(K, _case(dev, [(20, 4, 4)], 8, 2, 96, torch.float16, seed=19))
    with pytest.raises(NotImplementedError):
        _call(K, _case(dev, [(20, 4, 4)], 17, 1, 64, torch.float16, seed=19))


@pytest.mark.parametrize("n_q,nodes", [(8, 4), (16, 8), (32, 8)])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
def test_bad_drafts_in_many_short_sequences(cuda_device, n_q, nodes, D, dtype):
    """Every CTA runs through several sequences of one or two key tiles, most of them with a
    draft that holds an infinity: exactly the rows that see it carry it, every time.  The
    shapes have rows for one, two and four of a CTA's four softmax warps."""
    from vllm_mps_b200 import kernels as K

    rng = np.random.default_rng(n_q + D)
    seqs = []
    for _ in range(700):
        n = int(rng.integers(1, nodes + 1))
        seqs.append((int(rng.choice([0, 3, 20, 60])), n, n))
    seqs[0] = (60, nodes, nodes)
    c = _case(cuda_device, seqs, n_q, 2, D, dtype, seed=n_q, spare=float("nan"))
    want = _call(K, c)
    assert torch.isfinite(want).all()
    sees = torch.zeros(want.shape[0], dtype=torch.bool)
    mask, bt, at = c["mask"].cpu(), c["bt"].cpu(), 0
    blocks, slots = [], []
    for i, (ctx, n, _) in enumerate(seqs):
        if i % 5:  # the others stay as they are
            node = int(rng.integers(0, n))
            blocks.append(int(bt[i, (ctx + node) // 16]))
            slots.append((ctx + node) % 16)
            sees[at:at + n] = ((mask[at:at + n, 0] >> node) & 1).bool()
        at += n
    c["pool"][torch.tensor(blocks), 1, torch.tensor(slots), :, 5] = float("inf")
    expected = want.clone()
    expected[sees.to(cuda_device), :, 5] = float("inf")
    for _ in range(20):
        assert torch.equal(_call(K, c), expected)


@pytest.mark.parametrize("bits", [16.3, 20.05, 25.5])
@pytest.mark.parametrize("ctx", [200, 510, 8000])
@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 64)])
def test_many_small_weights_behind_a_large_one(cuda_device, ctx, bits, dtype, D):
    """One key holds the row, all others weigh 2^-bits of it and alone have a value.

    The bound of this file, and what a rounded weight may lose where the type runs out of
    exponents: an fp16 weight is at least 2^7 times its share of the largest, so half of
    its smallest step, 2^-25, is at most 2^-32 of the row's sum (bf16 has fp32's exponents).
    """
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(ctx, 1, 1)], 2, 1, D, dtype, seed=1)
    t = torch.arange(ctx + 1, device=cuda_device)
    blk = c["bt"][0, t // 16].long()
    c["q"].zero_()
    c["q"][..., 0] = 1.0
    pool = c["pool"]
    pool[blk, :, t % 16] = 0.0
    pool[blk, 0, t % 16, :, 0] = -bits * math.log(2)
    pool[blk, 1, t % 16] = 1.0
    pool[blk[3], :, 3] = 0.0
    got = _call(K, c, scale=1.0)
    out, big, mag = _reference(c, scale=1.0)
    lost = (ctx + 1) * 2.0 ** -32 if dtype == torch.float16 else 0.0
    tol = (2 * U[dtype] + 4 * D * 2.0 ** -23 * mag) * big + lost + U[dtype] * out.abs() + 1e-6
    assert ((got.double().cpu() - out).abs() <= tol).all()


def test_queries_as_a_matrix(cuda_device):
    """(total_q, n_q * D) queries, none of them included."""
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [(20, 4, 4)], 8, 2, 64, torch.float16, seed=20, q_pad=64)
    flat = torch.as_strided(c["q"], (4, 8 * 64), (c["q"].stride(0), 1))
    assert torch.equal(_call(K, dict(c, q=flat)), _call(K, c))
    c = _case(cuda_device, [(20, 0, 0)], 8, 2, 64, torch.float16, seed=20)
    assert _call(K, dict(c, q=c["q"].flatten(1))).shape == (0, 8, 64)
    with pytest.raises(ValueError):
        _call(K, dict(c, q=c["q"].flatten(1)[:, :500]))
