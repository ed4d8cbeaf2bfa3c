"""The host side of speculative decoding: tree topologies and the C ABI's refusals (no GPU)."""

import numpy as np
import pytest

from vllm_mps_b200.core.draft_tree import DraftTree


def _sees(mask, i, j):
    return bool((int(mask[i, j // 32]) >> (j % 32)) & 1)


def test_mask_holds_ancestors_and_self():
    rng = np.random.default_rng(0)
    for n in (1, 2, 31, 32, 33, 70):
        par = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
        t = DraftTree(par)
        m = t.mask()
        assert m.dtype == np.int32 and m.shape == (n, (n + 31) // 32)
        for i in range(n):
            anc, c = set(), i
            while c >= 0:
                anc.add(c)
                c = par[c]
            assert len(anc) - 1 == t.depths[i]
            for j in range(32 * m.shape[1]):
                assert _sees(m, i, j) == (j in anc)
        wide = t.mask(words=4)
        assert np.array_equal(wide[:, : m.shape[1]], m) and not wide[:, m.shape[1]:].any()


def test_widths_and_levels():
    t = DraftTree.from_widths((3, 2))
    assert t.parents.tolist() == [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3]
    assert t.level(0).tolist() == [0] and t.level(2).tolist() == [4, 5, 6, 7, 8, 9]
    assert t.max_depth == 2 and len(t) == 10


def test_refused_trees():
    for bad in ([], [-1, 1], [-1, -1], [-1, 0, 2]):
        with pytest.raises(ValueError):
            DraftTree(bad)
    with pytest.raises(ValueError):
        DraftTree.from_widths((2, 0))
    with pytest.raises(ValueError):
        DraftTree([-1] + [0] * 40).mask(words=1)


def test_host_side_refusals_need_no_gpu():
    from vllm_mps_b200 import kernels as K

    lib = K.load_library()
    base = 1 << 20  # never dereferenced on these paths
    tree = lambda **kw: lib.vmps_paged_tree_attention(  # noqa: E731
        kw.get("out", base), kw.get("q", base), kw.get("qs", 8 * 64), base, base, kw.get("mb", 4),
        base, base, base, base, base, kw.get("words", 1), kw.get("seqs", 2), kw.get("rows", 4),
        kw.get("max_q", 2), kw.get("n_q", 8), kw.get("n_kv", 2), kw.get("d", 64),
        kw.get("bs", 16), kw.get("nb", 10), kw.get("scale", 0.125), None, 0, kw.get("dt", 0), None)
    assert tree(dt=3) == -1 and b"dtype" in lib.vmps_last_error()
    assert tree(words=0) == -1
    assert tree(d=96) == -2
    assert tree(bs=32) == -2 and b"block_size" in lib.vmps_last_error()
    assert tree(n_q=34) == -2   # 17 query heads per kv head
    assert tree(n_q=9) == -2
    assert tree(seqs=5000) == -2
    assert tree(q=None) == -1
    assert tree(q=base + 8) == -3
    assert tree(qs=500) == -3
    assert tree(qs=256) == -1
    assert tree(scale=0.0) == -1
    assert tree(seqs=0) == 0 and tree(rows=0) == 0 and tree(max_q=0) == 0
    commit = lambda **kw: lib.vmps_commit_tree(  # noqa: E731
        base, base, base, kw.get("pool", base), kw.get("layers", 1), base, 4, base, base, base,
        base, base, base, kw.get("seqs", 2), 10, kw.get("max_tree", 5), kw.get("n_kv", 2),
        kw.get("d", 64), kw.get("bs", 16), 10, kw.get("dt", 0), None)
    assert commit(layers=0) == -1
    assert commit(dt=9) == -1
    assert commit(bs=8) == -2
    assert commit(max_tree=1025) == -2
    assert commit(n_kv=1, d=4) == -2
    assert commit(pool=None) == -1
    assert commit(pool=base + 2) == -3
    assert commit(seqs=0) == 0
    assert lib.vmps_w4_gemm_supported(32, 7, 96, 32) == 1
    assert lib.vmps_w4_gemm_supported(33, 7, 96, 32) == 0
    assert lib.vmps_w4_gemm_supported(1, 7, 96, 64) == 0
    assert lib.vmps_w4_gemm_supported(1, 7, 96, 48) == 0
    w4 = lambda **kw: lib.vmps_w4_gemm(  # noqa: E731
        kw.get("out", base), kw.get("os", 64), kw.get("x", base), kw.get("xs", 128), base, base,
        kw.get("z", None), kw.get("m", 2), 64, 128, 64, 0, kw.get("dt", 0), None)
    assert w4(dt=2) == -1
    assert w4(m=40) == -2 and b"M=40" in lib.vmps_last_error()
    assert w4(x=None) == -1
    assert w4(xs=120) == -1 and w4(os=60) == -1
    assert w4(x=base + 8) == -3 and w4(z=base + 4) == -3 and w4(xs=132) == -3
    assert w4(out=base + 1) == -3
    assert w4(m=0) == 0
