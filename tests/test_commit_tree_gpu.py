"""Commit of an accepted branch: the walk, and K/V moved in every layer, exactly."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _walk(parents, tokens, target):
    path = [0]
    while True:
        cur = path[-1]
        nxt = [c for c in range(cur + 1, len(parents))
               if parents[c] == cur and tokens[c] == target[cur]]
        if not nxt:
            return path
        path.append(nxt[0])


def _case(dev, ctx, sizes, layers, n_kv, D, dtype, seed, agree=0.8, vocab=6):
    """Few token values, so that siblings with equal tokens and chance matches occur."""
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in zip(ctx, sizes)]
    pages = [(x + 15) // 16 for x in lens]
    order = rng.permutation(sum(pages) + 2)
    bt = np.zeros((len(ctx), max(1, max(pages))), np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = order[at:at + n]
        at += n
    trees = []
    for n in sizes:
        par = [-1] + [int(rng.integers(max(0, (i - 1) // 2), i)) for i in range(1, n)]
        tok = rng.integers(0, vocab, size=n)
        tgt = rng.integers(0, vocab, size=n)
        for i in range(n):
            kids = [c for c in range(n) if c and par[c] == i]
            if kids and rng.random() < agree:
                tgt[i] = tok[kids[int(rng.integers(len(kids)))]]
        trees.append((par[:n], tok.tolist(), tgt.tolist()))
    g = torch.Generator(device=dev).manual_seed(seed)
    pool = torch.randn((layers, len(order), 2, 16, n_kv, D), generator=g, device=dev).to(dtype)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    flat = lambda j: [x for t in trees for x in t[j]]  # noqa: E731
    cu = np.cumsum([0] + list(sizes))[:-1]
    return dict(pool=pool, bt=i32(bt), ctx=i32(ctx), lens=i32(lens), cu=i32(cu), par=i32(flat(0)),
                tok=i32(flat(1)), tgt=torch.tensor(flat(2), dtype=torch.int64, device=dev),
                max_tree=max(1, max(sizes)), trees=trees, at=ctx, tables=bt)


def _call(K, c, pool=None):
    return K.commit_tree(c["pool"] if pool is None else pool, c["bt"], c["ctx"], c["lens"], c["cu"],
                         c["par"], c["tok"], c["tgt"], c["max_tree"])


def _check(c, before, got):
    path, count, nxt = (x.cpu() for x in got)
    want = before.clone()
    for i, (par, tok, tgt) in enumerate(c["trees"]):
        p = _walk(par, tok, tgt) if par else []
        assert count[i] == len(p)
        assert path[i].tolist() == p + [-1] * (c["max_tree"] - len(p))
        assert nxt[i] == (tgt[p[-1]] if p else -1)
        for k, node in enumerate(p):
            s, d = c["at"][i] + node, c["at"][i] + k
            bs, bd = int(c["tables"][i][s // 16]), int(c["tables"][i][d // 16])
            want[:, bd, :, d % 16] = before[:, bs, :, s % 16]
    return want


CASES = [
    # ctx, sizes, layers, n_kv, D
    ([86], [8], 22, 4, 64),
    ([0, 15, 16, 31, 100], [1, 2, 20, 33, 64], 3, 8, 128),
    ([5] * 40, list(range(1, 41)), 2, 1, 64),
    ([7, 1], [500, 300], 1, 2, 64),
    ([14, 2, 9], [26, 0, 12], 4, 3, 8),       # an empty tree between others
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_walk_and_moves(cuda_device, case, dtype):
    from vllm_mps_b200 import kernels as K

    ctx, sizes, layers, n_kv, D = CASES[case]
    for agree in (0.0, 0.8, 1.0):
        c = _case(cuda_device, ctx, sizes, layers, n_kv, D, dtype, seed=case, agree=agree)
        before = c["pool"].cpu()
        got = _call(K, c)
        want = _check(c, before, got)
        assert torch.equal(c["pool"].cpu(), want)  # and nothing else was touched


def test_long_branch_moves_in_order(cuda_device):
    """A path whose targets are later sources: every other node of a chain of pairs."""
    from vllm_mps_b200 import kernels as K

    n = 61
    par = [-1] + [max(0, ((i - 1) // 2) * 2) for i in range(1, n)]
    tok = list(range(n))
    tgt = [i + 2 if i % 2 == 0 and i + 2 < n else -5 for i in range(n)]
    c = _case(cuda_device, [10], [n], 2, 2, 64, torch.float16, seed=1)
    c["trees"] = [(par, tok, tgt)]
    for key, v in (("par", par), ("tok", tok), ("tgt", tgt)):
        c[key].copy_(torch.tensor(v))
    before = c["pool"].cpu()
    got = _call(K, c)
    want = _check(c, before, got)
    assert int(got[1][0]) == 31
    assert torch.equal(c["pool"].cpu(), want)


def test_single_layer_pool_and_special_values(cuda_device):
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [30, 4], [12, 9], 1, 2, 64, torch.float16, seed=4, agree=1.0)
    c["pool"].view(torch.int16).random_(-2 ** 15, 2 ** 15)  # NaN and infinity patterns move as bits
    before = c["pool"].cpu()
    got = _call(K, c, pool=c["pool"][0])
    want = _check(c, before, got)
    assert torch.equal(c["pool"].cpu().view(torch.int16), want.view(torch.int16))


def test_bad_indices_are_reported_and_skipped(cuda_device):
    from vllm_mps_b200 import kernels as K

    dev = cuda_device
    c = _case(dev, [10, 20, 30], [12, 12, 12], 2, 2, 64, torch.float16, seed=6, agree=1.0)
    before = c["pool"].clone()
    good = [x.clone() for x in _call(K, c)]
    after = c["pool"].clone()
    # A tree outside the given rows counts as empty.
    cu = c["cu"].clone()
    cu[1] = 30
    pool = before.clone()
    path, count, nxt = _call(K, dict(c, cu=cu), pool=pool)
    assert K.error_word(dev) & 64
    assert int(count[1]) == 0 and int(nxt[1]) == -1 and (path[1] == -1).all()
    assert torch.equal(path[0], good[0][0]) and torch.equal(path[2], good[0][2])
    # A block id outside the pool: that slot is not moved, the other sequences are.
    bt = c["bt"].clone()
    bt[1, :] = 10 ** 6
    pool = before.clone()
    _call(K, dict(c, bt=bt), pool=pool)
    assert K.error_word(dev) & 2
    for i in (0, 2):
        ids = c["bt"][i, : (c["at"][i] + 12 + 15) // 16].long()
        assert torch.equal(pool[:, ids], after[:, ids])


def test_refusals(cuda_device):
    from vllm_mps_b200 import kernels as K

    c = _case(cuda_device, [10], [5], 2, 2, 64, torch.float16, seed=7)
    with pytest.raises(TypeError):
        _call(K, dict(c, tgt=c["tgt"].int()))
    with pytest.raises(TypeError):
        _call(K, dict(c, tok=c["tok"].long()))
    with pytest.raises(ValueError):
        _call(K, dict(c, par=c["par"][:3]))
    with pytest.raises(ValueError):
        _call(K, dict(c, max_tree=0))
    with pytest.raises(NotImplementedError):
        _call(K, dict(c, max_tree=1025))
    with pytest.raises(ValueError):
        _call(K, c, pool=c["pool"].transpose(3, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        _call(K, dict(c, tok=c["tok"].cpu()))
