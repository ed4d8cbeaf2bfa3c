"""Timing cases of the speculative-decoding operators: tree attention over the paged
cache, the commit of an accepted branch, and products with 4-bit weights.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same
ranges, ``prepare`` builds what a caller holds before the call, ``run`` makes
one pass and ``exact`` computes the same outputs in 64 bits.  With ``own``
false, ``run`` is the plain form: elementary torch operations in fp32,
rounded once at the end.  With ``own`` true it calls the framework's kernels.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _dev():
    return torch.device("cuda")


# ── cases ────────────────────────────────────────────────────────────────────


def listed():
    return [
        # One short chat turn on a small model: a tree of 8 drafts, latency only.
        dict(name="tree one short", op="tree", seqs=1, ctx_lo=137, ctx=137, nodes=8, nodes_lo=8,
             rows=0, n_q=32, n_kv=4, d=64, dtype="f16"),
        # Plain decoding through the same call: one token per sequence, ragged prompts.
        dict(name="tree single token", op="tree", seqs=24, ctx_lo=1, ctx=2048, nodes=1, nodes_lo=1,
             rows=0, n_q=32, n_kv=4, d=64, dtype="f16"),
        # A serving batch, ragged contexts, trees of up to 26 nodes checked at once.
        dict(name="tree batch check", op="tree", seqs=32, ctx_lo=1, ctx=4096, nodes=26, nodes_lo=5,
             rows=0, n_q=32, n_kv=8, d=128, dtype="bf16"),
        # The last level of a tree being drafted: 4 query rows, 13 drafts already cached.
        dict(name="tree draft level", op="tree", seqs=4, ctx_lo=3001, ctx=16383, nodes=17, nodes_lo=17,
             rows=4, n_q=32, n_kv=8, d=128, dtype="bf16"),
        # Four long documents (the 131072-token context of the decode benchmark), 16 nodes.
        dict(name="tree long contexts", op="tree", seqs=4, ctx_lo=131072, ctx=131072, nodes=16,
             nodes_lo=16, rows=0, n_q=32, n_kv=8, d=128, dtype="bf16"),
        # Wide trees on a model with 8 query heads per kv head: bound by arithmetic.
        dict(name="tree wide check", op="tree", seqs=8, ctx_lo=5003, ctx=8192, nodes=64, nodes_lo=64,
             rows=0, n_q=64, n_kv=8, d=128, dtype="bf16"),
        # The small model's fused QKV projection for one drafted token.
        dict(name="w4 small qkv", op="w4", m=1, n=2560, k=2048, group=128, zeros=False, silu=False,
             dtype="f16"),
        # The 8B model's gate and up projections with the activation, one token.
        dict(name="w4 gate up", op="w4", m=1, n=14336, k=4096, group=128, zeros=True, silu=True,
             dtype="bf16"),
        # Its down projection for a level of 5 nodes, finer groups.
        dict(name="w4 down level", op="w4", m=5, n=4096, k=14336, group=64, zeros=True, silu=False,
             dtype="bf16"),
        # Its LM head for 4 sequences x 4 drafts.
        dict(name="w4 lm head", op="w4", m=16, n=128256, k=4096, group=128, zeros=False, silu=False,
             dtype="bf16"),
        # One sequence's accepted branch, 22 layers of the small model.
        dict(name="commit one", op="commit", seqs=1, ctx_lo=86, ctx=86, nodes=8, nodes_lo=8,
             layers=22, n_kv=4, d=64, dtype="f16"),
        # A batch of 64 ragged trees on 32 layers.
        dict(name="commit batch", op="commit", seqs=64, ctx_lo=1, ctx=128, nodes=26, nodes_lo=3,
             layers=32, n_kv=8, d=128, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "w4", "w4", "commit"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "tree":
        d = rng.choice([64, 128])
        n_kv = rng.choice([1, 2, 4, 8, 16])
        n_q = n_kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        nodes = _log(rng, 1, 64)
        while True:
            seqs, ctx = _log(rng, 1, 64), _log(rng, 1, 131072)
            rows = min(nodes, rng.choice([nodes, nodes, _log(rng, 1, 8)]))
            cost = seqs * (ctx + nodes) * d
            if cost * n_kv <= 4 * 131072 * 8 * 128 and cost * n_q * rows <= 8 * 8192 * 128 * 64 * 64:
                break
        return dict(op="tree", seqs=seqs, ctx_lo=rng.choice([1, ctx, max(1, ctx // 3)]), ctx=ctx,
                    nodes=nodes, nodes_lo=rng.choice([nodes, max(1, nodes // 4)]),
                    rows=0 if rows == nodes else rows, n_q=n_q, n_kv=n_kv, d=d, dtype=dtype)
    if op == "w4":
        group = rng.choice([32, 64, 128])
        silu = rng.random() < 0.3
        while True:
            n, k = _log(rng, 256, 65536), group * _log(rng, 512 // group, 16384 // group)
            if n * k * (2 if silu else 1) <= 128256 * 4096:
                break
        return dict(op="w4", m=_log(rng, 1, 32), n=n, k=k, group=group, zeros=rng.random() < 0.5,
                    silu=silu, dtype=dtype)
    ctx = _log(rng, 1, 128)
    return dict(op="commit", seqs=_log(rng, 1, 64), ctx_lo=rng.choice([1, ctx]), ctx=ctx,
                nodes=_log(rng, 1, 64), nodes_lo=1, layers=_log(rng, 1, 32),
                n_kv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128]), dtype=dtype)


# ── what follows from a case alone (lengths, topologies, which drafts are accepted) ──


def _shape_rng(case):
    return random.Random("|".join("%s=%s" % kv for kv in sorted(case.items()) if kv[0] != "name"))


def _tree(rng, n):
    """Parents of a tree of n nodes, numbered so that a parent comes before its children."""
    par = [-1]
    for i in range(1, n):
        lo = (i - 1) // 3
        par.append(rng.randint(lo, min(i - 1, lo + 2)))
    return par


def _plan(case):
    """Context lengths and parents of every sequence; which child, if any, the model picks."""
    rng = _shape_rng(case)
    ctx = [rng.randint(case["ctx_lo"], case["ctx"]) for _ in range(case["seqs"])]
    ctx[0] = case["ctx"]
    sizes = [rng.randint(case["nodes_lo"], case["nodes"]) for _ in range(case["seqs"])]
    sizes[0] = case["nodes"]
    trees = [_tree(rng, n) for n in sizes]
    picks = []
    for par in trees:
        kids = [[c for c in range(len(par)) if par[c] == i] for i in range(len(par))]
        picks.append([rng.choice(k) if k and rng.random() < 0.85 else -1 for k in kids])
    return ctx, trees, picks


def _paths(trees, picks):
    out = []
    for par, pick in zip(trees, picks):
        path, cur = [0], 0
        while pick[cur] >= 0:
            cur = pick[cur]
            path.append(cur)
        out.append(path)
    return out


def _mask_rows(par):
    """Ancestor sets (the node itself included) as Python integers."""
    rows = []
    for i, p in enumerate(par):
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
    return rows


def _mask_words(trees, keep):
    words = max(1, max((len(t) + 31) // 32 for t in trees))
    rows = []
    for par, q in zip(trees, keep):
        for r in _mask_rows(par)[len(par) - q:]:
            rows.append([(r >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
    return np.array(rows, dtype=np.uint32).reshape(-1, words).view(np.int32)


def _tables(rng, lens):
    """Block tables over a shuffled pool with a few spare blocks."""
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    order = rng.permutation(sum(pages) + 3)
    bt = np.zeros((len(lens), max(1, max(pages))), dtype=np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = order[at:at + n]
        at += n
    return bt, sum(pages) + 3


def _starts(sizes):
    return [sum(sizes[:i]) for i in range(len(sizes))]


# ── inputs ───────────────────────────────────────────────────────────────────


def prepare(case, seed):
    g = torch.Generator(device=_dev())
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=_dev(), dtype=dtype)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=_dev())

    if case["op"] == "w4":
        n, k, m = case["n"] * (2 if case["silu"] else 1), case["k"], case["m"]
        ng = k // case["group"]
        codes = torch.randint(0, 256, (n, k // 2), generator=g, device=_dev(), dtype=torch.uint8)
        spread = 0.5 + torch.rand((n, ng), generator=g, device=_dev())
        scales = (spread / (4.6 * math.sqrt(k))).to(dt)
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(5, 12, (n, ng), generator=g, device=_dev(), dtype=torch.uint8)
        s = dict(case=case, x=randn(m, k), codes=codes, scales=scales, zeros=zeros)
        return s

    ctx, trees, picks = _plan(case)
    total = [c + len(t) for c, t in zip(ctx, trees)]
    bt, nblk = _tables(rng, total)
    s = dict(case=case, bt=torch.from_numpy(bt).to(_dev()), ctx=i32(ctx), seq_lens=i32(total),
             parents=i32([p for t in trees for p in t]))
    n_kv, d = case["n_kv"], case["d"]
    if case["op"] == "tree":
        keep = [len(t) if not case["rows"] else min(case["rows"], len(t)) for t in trees]
        s["pool"] = randn(nblk, 2, PAGE, n_kv, d)
        s["qkv"] = randn(sum(keep), (case["n_q"] + 2 * n_kv) * d) * 1.5
        s["q"] = s["qkv"][:, : case["n_q"] * d].unflatten(1, (case["n_q"], d))
        s["mask"] = torch.from_numpy(_mask_words(trees, keep)).to(_dev())
        s["q_lens"], s["cu_q"], s["max_q"] = i32(keep), i32(_starts(keep)), max(keep)
        return s
    sizes = [len(t) for t in trees]
    vocab = 32000
    tokens, target = [], []
    for par, pick in zip(trees, picks):
        # Siblings carry different tokens, as the best continuations of a node do.
        tok = rng.integers(0, vocab, size=len(par))
        for i, p in enumerate(par):
            taken = {int(tok[c]) for c in range(i) if par[c] == p}
            while p >= 0 and int(tok[i]) in taken:
                tok[i] = (tok[i] + 1) % vocab
        for i, p in enumerate(pick):
            other = int(rng.integers(vocab, 2 * vocab))  # not among the drafts
            target.append(int(tok[p]) if p >= 0 else other)
        tokens += tok.tolist()
    s["pool"] = randn(case["layers"], nblk, 2, PAGE, n_kv, d)
    s["tokens"] = i32(tokens)
    s["target"] = torch.tensor(target, dtype=torch.int64, device=_dev())
    s["cu_tree"], s["max_tree"] = i32(_starts(sizes)), max(sizes)
    s["mask"] = torch.from_numpy(_mask_words(trees, sizes)).to(_dev())
    return s


# ── one pass ─────────────────────────────────────────────────────────────────


def run(state):
    op = state["case"]["op"]
    if own:
        from vllm_mps_b200 import kernels as K

        if op == "tree":
            return K.paged_tree_attention(state["q"], state["pool"], state["bt"], state["ctx"],
                                          state["seq_lens"], state["q_lens"], state["cu_q"],
                                          state["mask"], state["max_q"])
        if op == "w4":
            w = K.W4Weight(state["codes"], state["scales"], state["zeros"])
            return K.w4_gemm(state["x"], w, silu_mul=state["case"]["silu"])
        path, count, nxt = K.commit_tree(state["pool"], state["bt"], state["ctx"],
                                         state["seq_lens"], state["cu_tree"], state["parents"],
                                         state["tokens"], state["target"], state["max_tree"])
        return dict(path=path, count=count, next=nxt, pool=state["pool"])
    return {"tree": _plain_tree, "w4": _plain_w4, "commit": _plain_commit}[op](state)


def _bits(mask, width):
    """(rows, words) int32 -> (rows, width) truth values."""
    j = torch.arange(width, device=mask.device)
    word = mask[:, torch.clamp(j // 32, max=mask.shape[1] - 1)]
    return ((word >> (j % 32)) & 1).bool()


def _plain_tree(s):
    q, pool, bt = s["q"], s["pool"], s["bt"].long()
    dev = q.device
    B, P = bt.shape
    n_kv, d = pool.shape[3], pool.shape[4]
    G = q.shape[1] // n_kv
    R, L = s["max_q"], P * PAGE
    kv = pool[bt]
    k = kv[:, :, 0].reshape(B, L, n_kv, d).permute(0, 2, 3, 1).float()
    v = kv[:, :, 1].reshape(B, L, n_kv, d).permute(0, 2, 1, 3).float()
    r = torch.arange(R, device=dev)
    live = r < s["q_lens"].unsqueeze(1)
    row = torch.where(live, s["cu_q"].unsqueeze(1) + r, 0).long()
    qr = q[row].float().view(B, R, n_kv, G, d).permute(0, 2, 1, 3, 4).reshape(B, n_kv, R * G, d)
    t = torch.arange(L, device=dev)
    ctx, end = s["ctx"].long()[:, None, None], s["seq_lens"].long()[:, None, None]
    width = int(s["mask"].shape[1]) * 32
    bits = _bits(s["mask"], width)[row]
    drafted = bits.gather(2, (t - ctx).clamp(0, width - 1).expand(B, R, L))
    see = (t < end) & ((t < ctx) | drafted) & live.unsqueeze(2)
    see = see.repeat_interleave(G, 1).unsqueeze(1)
    x = torch.matmul(qr, k) * (1.0 / math.sqrt(d))
    x = torch.where(see, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(l == 0, 1.0, l)
    o = o.view(B, n_kv, R, G, d).permute(0, 2, 1, 3, 4).reshape(B, R, n_kv * G, d)
    return o[live].to(q.dtype)


def _plain_w4(s):
    x, codes, scales = s["x"], s["codes"], s["scales"]
    q = torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1).float()
    ng = scales.shape[1]
    z = 8.0 if s["zeros"] is None else s["zeros"].float().unsqueeze(2)
    w = (q.view(q.shape[0], ng, -1) - z) * scales.float().unsqueeze(2)
    y = torch.matmul(x.float(), w.view(q.shape).t())
    if s["case"]["silu"]:
        a, b = y.chunk(2, 1)
        y = a / (1.0 + torch.exp(-a)) * b
    return y.to(x.dtype)


def _plain_commit(s):
    pool, bt = s["pool"], s["bt"].long()
    dev = pool.device
    B, n = bt.shape[0], s["max_tree"]
    ctx = s["ctx"].long()
    size = s["seq_lens"].long() - ctx
    i = torch.arange(n, device=dev)
    live = i < size.unsqueeze(1)
    row = torch.where(live, s["cu_tree"].unsqueeze(1) + i, 0).long()
    par = torch.where(live, s["parents"][row].long(), -1)
    tok = s["tokens"].long()[row]
    tgt = s["target"][row]
    good = (tok == tgt.gather(1, par.clamp(min=0))) & (par >= 0) & live
    # Of several children with the same token the lowest-numbered one counts.
    twin = (par.unsqueeze(2) == par.unsqueeze(1)) & good.unsqueeze(2) & good.unsqueeze(1)
    good = good & ~(twin & (i.unsqueeze(0) < i.unsqueeze(1))).any(2)
    good[:, 0] = size > 0
    anc = _bits(s["mask"], n)[row]
    taken = ~(anc & ~good.unsqueeze(1)).any(2) & live
    count = taken.sum(1)
    order = torch.where(taken, i, n).sort(1).values
    path = torch.where(order < n, order, -1)
    last = path.gather(1, (count - 1).clamp(min=0).unsqueeze(1))
    nxt = torch.where(count > 0, tgt.gather(1, last.clamp(min=0)).squeeze(1), -1)
    move = (path >= 0) & (path != i)
    b, k = move.nonzero(as_tuple=True)
    src, dst = ctx[b] + path[b, k], ctx[b] + k
    kv = pool[:, bt[b, src // PAGE], :, src % PAGE]
    pool[:, bt[b, dst // PAGE], :, dst % PAGE] = kv
    return dict(path=path.int(), count=count.int(), next=nxt, pool=pool)


# ── the same in 64 bits, from the definitions ────────────────────────────────


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "commit":
        return None  # nothing is computed but whole numbers and copies
    if case["op"] == "w4":
        x = s["x"].double()
        outs = []
        step = 8192
        for at in range(0, s["codes"].shape[0], step):
            c = s["codes"][at:at + step]
            w = torch.empty((c.shape[0], case["k"]), dtype=torch.float64, device=c.device)
            w[:, 0::2] = (c % 16).double()
            w[:, 1::2] = (c // 16).double()
            for j in range(s["scales"].shape[1]):
                part = w[:, j * case["group"]:(j + 1) * case["group"]]
                part -= 8 if s["zeros"] is None else s["zeros"][at:at + step, j:j + 1].double()
                part *= s["scales"][at:at + step, j:j + 1].double()
            outs.append(torch.einsum("mk,nk->mn", x, w))
        y = torch.cat(outs, 1)
        if case["silu"]:
            a, b = y[:, : case["n"]], y[:, case["n"]:]
            y = a * torch.sigmoid(a) * b
        return y
    ctx, trees, _ = _plan(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    G = case["n_q"] // case["n_kv"]
    at = 0
    for i, (c, par) in enumerate(zip(ctx, trees)):
        n = len(par)
        q_len = int(s["q_lens"][i])
        ids = s["bt"][i, : (c + n + PAGE - 1) // PAGE].long()
        see = torch.ones((q_len, c + n), dtype=torch.bool)
        for r, bits in enumerate(_mask_rows(par)[n - q_len:]):
            see[r, c:] = torch.tensor([(bits >> j) & 1 for j in range(n)], dtype=torch.bool)
        see = see.to(out.device)
        for h in range(case["n_kv"]):
            k = s["pool"][ids, 0, :, h].flatten(0, 1)[: c + n].double()
            v = s["pool"][ids, 1, :, h].flatten(0, 1)[: c + n].double()
            qh = s["q"][at:at + q_len, h * G:(h + 1) * G].double()
            x = torch.einsum("rgd,td->rgt", qh, k) / math.sqrt(case["d"])
            p = torch.softmax(x.masked_fill(~see.unsqueeze(1), float("-inf")), -1)
            out[at:at + q_len, h * G:(h + 1) * G] = torch.einsum("rgt,td->rgd", p, v)
        at += q_len
    return out


# ── what a pass cannot do without ────────────────────────────────────────────


def work(case):
    if case["op"] == "w4":
        n, k, m = case["n"] * (2 if case["silu"] else 1), case["k"], case["m"]
        side = n * (k // case["group"]) * (3 if case["zeros"] else 2)
        return dict(bytes=n * k // 2 + side + 2 * m * (k + case["n"]), flops=2 * m * n * k)
    ctx, trees, picks = _plan(case)
    row = 2 * case["n_kv"] * case["d"]  # bytes of one token's K (or V)
    if case["op"] == "commit":
        moved = sum(1 for p in _paths(trees, picks) for i, x in enumerate(p) if i != x)
        nodes = sum(len(t) for t in trees)
        return dict(bytes=moved * case["layers"] * 2 * row * 2 + nodes * 16 + case["seqs"] * 64,
                    flops=0)
    data = flops = 0
    for c, par in zip(ctx, trees):
        q = len(par) if not case["rows"] else min(case["rows"], len(par))
        seen = sum(bin(r).count("1") for r in _mask_rows(par)[len(par) - q:])
        data += 2 * (c + len(par)) * row + 2 * q * case["n_q"] * case["d"] * 2 + 8 * q
        flops += 4 * case["n_q"] * case["d"] * (q * c + seen)
    return dict(bytes=data, flops=flops)
