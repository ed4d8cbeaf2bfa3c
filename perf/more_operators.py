"""Timing cases of the 8-bit paged cache: norms and rotation of queries and keys with the
cache write, the cache's read-back, and decode attention over it.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same
ranges, ``prepare`` builds what a caller holds before the call, ``run`` makes
one pass and ``exact`` computes the same outputs in 64 bits.  With ``own``
false, ``run`` is the plain form: elementary torch operations in fp32 (angles
in 64 bits), rounded once at the end.  With ``own`` true it calls the
framework's kernels.

The cache: ``codes`` (num_blocks, 2, 16, n_kv, d), int8 or e4m3, and ``scales``
(num_blocks, n_kv, 2, 16) fp32; a stored value is code * scale.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
EPS = 1e-6
TINY = 2.0 ** -100  # rows below it are stored as zeros
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_FMT = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}


def _dev():
    return torch.device("cuda")


# ── cases ────────────────────────────────────────────────────────────────────


def listed():
    return [
        # One token of one chat on the 8B-sized layer, norms on, 16-bit cache: latency only.
        dict(name="norm rope one token", op="store", seqs=1, lo=1024, hi=1024, rows=1, norm=True,
             n_q=32, n_kv=8, d=128, dtype="bf16", fmt="none"),
        # A decode step of 64 ragged sequences on the small model, 16-bit cache.
        dict(name="norm rope decode batch", op="store", seqs=64, lo=1, hi=2048, rows=1, norm=True,
             n_q=32, n_kv=4, d=64, dtype="f16", fmt="none"),
        # Ragged prompts of the small model into the int8 cache, then read back for their attention.
        dict(name="prompts int8", op="store", seqs=16, lo=1, hi=256, rows=0, norm=False,
             n_q=32, n_kv=4, d=64, dtype="f16", fmt="int8"),
        # A full prefill chunk (8192 rows) of the 8B-sized layer into the e4m3 cache, and back.
        dict(name="prompt chunk fp8", op="store", seqs=4, lo=2048, hi=2048, rows=0, norm=True,
             n_q=32, n_kv=8, d=128, dtype="bf16", fmt="fp8"),
        # Contexts of a ragged batch read back before the next chunk of their prompts.
        dict(name="read ragged int8", op="read", seqs=24, lo=1, hi=2048, n_kv=4, d=64, dtype="f16",
             fmt="int8"),
        # One long document's context read back.
        dict(name="read long fp8", op="read", seqs=1, lo=131071, hi=131071, n_kv=8, d=128,
             dtype="bf16", fmt="fp8"),
        # One short chat turn on the small model: latency only.
        dict(name="decode one short", op="decode", seqs=1, lo=137, hi=137, n_q=32, n_kv=4, d=64,
             dtype="f16", fmt="int8"),
        # The decode benchmark's batch: 64 sequences, contexts spread over 1..2048.
        dict(name="decode ragged batch", op="decode", seqs=64, lo=1, hi=2048, n_q=32, n_kv=4, d=64,
             dtype="f16", fmt="int8"),
        # A serving batch on the 8B-sized layer in e4m3.
        dict(name="decode batch fp8", op="decode", seqs=32, lo=1, hi=4096, n_q=32, n_kv=8, d=128,
             dtype="bf16", fmt="fp8"),
        # Four long documents (the decode benchmark's 131072-token contexts).
        dict(name="decode long contexts", op="decode", seqs=4, lo=131072, hi=131072, n_q=32, n_kv=8,
             d=128, dtype="bf16", fmt="int8"),
        # One kv head shared by 16 query heads, odd lengths.
        dict(name="decode one kv head", op="decode", seqs=7, lo=9001, hi=16383, n_q=16, n_kv=1,
             d=128, dtype="bf16", fmt="fp8"),
        # A large batch of medium contexts, 8 query heads a kv head.
        dict(name="decode wide batch", op="decode", seqs=256, lo=511, hi=1537, n_q=64, n_kv=8, d=128,
             dtype="bf16", fmt="int8"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "store", "read", "decode", "decode", "decode"])
    d = rng.choice([64, 128])
    n_kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    n_q = n_kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    case = dict(op=op, n_kv=n_kv, d=d, dtype=rng.choice(["f16", "bf16"]))
    if op == "store":
        rows = rng.choice([0, 0, 1])
        while True:
            seqs, hi = _log(rng, 1, 256), _log(rng, 1, 8192)
            if (seqs if rows else seqs * hi) * (n_q + 2 * n_kv) * d <= 8192 * 48 * 128 \
                    and seqs * hi * n_kv * d <= 64 * 2048 * 8 * 128:
                break
        fmt = "none" if rows else rng.choice(["int8", "fp8"])
        return dict(case, seqs=seqs, lo=rng.choice([1, hi, max(1, hi // 3)]), hi=hi, rows=rows,
                    norm=rng.random() < 0.6, n_q=n_q, fmt=fmt)
    most = 131071 * 8 * 128 if op == "read" else 4 * 131072 * 8 * 128
    while True:
        seqs, hi = _log(rng, 1, 256), _log(rng, 1, 131072)
        if seqs * hi * n_kv * d <= most:
            break
    case = dict(case, seqs=seqs, lo=rng.choice([1, hi, max(1, hi // 3)]), hi=hi,
                fmt=rng.choice(["int8", "fp8"]))
    return case if op == "read" else dict(case, n_q=n_q)


# ── what follows from a case alone ───────────────────────────────────────────


def _lens(case):
    rng = random.Random("|".join("%s=%s" % kv for kv in sorted(case.items()) if kv[0] != "name"))
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    lens[0] = case["hi"]
    return lens


def _rows(case, lens):
    """(sequence, position) of every new row: the last token of each, or all of them."""
    if case["rows"]:
        return list(range(len(lens))), [n - 1 for n in lens]
    seq = np.repeat(np.arange(len(lens)), lens)
    first = np.repeat(np.cumsum([0] + lens[:-1]), lens)
    return seq.tolist(), (np.arange(len(seq)) - first).tolist()


def _tables(rng, lens):
    """Block tables over a shuffled pool with a few spare blocks."""
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    order = rng.permutation(sum(pages) + 3)
    bt = np.zeros((len(lens), max(pages)), dtype=np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = order[at:at + n]
        at += n
    return bt, len(order)


def _packed(lens):
    """Tables of a pool that holds the sequences' pages one after the other."""
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    bt = np.zeros((len(lens), max(pages)), dtype=np.int32)
    at = 0
    for i, n in enumerate(pages):
        bt[i, :n] = np.arange(at, at + n)
        at += n
    return bt, at


# ── inputs ───────────────────────────────────────────────────────────────────


def prepare(case, seed):
    g = torch.Generator(device=_dev())
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = _DT[case["dtype"]]
    n_kv, d = case["n_kv"], case["d"]

    def i32(v):
        return torch.from_numpy(np.asarray(v, dtype=np.int32)).to(_dev())

    def randn(*shape):
        return torch.randn(shape, generator=g, device=_dev(), dtype=dt)

    lens = _lens(case)
    bt, blocks = _tables(rng, lens)
    # Keys have channels that are larger in every token.
    gain = 1.0 + 5.0 * (torch.rand((n_kv, d), generator=g, device=_dev()) < 0.03)
    s = dict(case=case, bt=i32(bt), lens=i32(lens))
    if case["op"] == "store":
        seq, pos = _rows(case, lens)
        n_q, rows = case["n_q"], len(pos)
        seq, at = np.asarray(seq), np.asarray(pos)
        s["qkv"] = randn(rows, (n_q + 2 * n_kv) * d)
        s["qkv"][:, n_q * d:(n_q + n_kv) * d] *= gain.flatten()
        s["positions"], s["slots"] = i32(at), i32(bt[seq, at // PAGE] * PAGE + at % PAGE)
        s["inv_freq"] = (1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(_dev())
        s["q_weight"] = (1.0 + 0.1 * randn(d)).to(dt) if case["norm"] else None
        s["k_weight"] = (1.0 + 0.1 * randn(d)).to(dt) if case["norm"] else None
        if case["fmt"] == "none":
            s["pool"] = randn(blocks, 2, PAGE, n_kv, d)
            return s
        s["codes"] = torch.zeros((blocks, 2, PAGE, n_kv, d), device=_dev(), dtype=_FMT[case["fmt"]][0])
        s["scales"] = torch.zeros((blocks, n_kv, 2, PAGE), device=_dev())
    else:
        s["codes"] = torch.empty((blocks, 2, PAGE, n_kv, d), device=_dev(), dtype=_FMT[case["fmt"]][0])
        s["scales"] = torch.empty((blocks, n_kv, 2, PAGE), device=_dev())
        step = max(1, (1 << 26) // (2 * PAGE * n_kv * d))
        for i in range(0, blocks, step):
            x = randn(min(step, blocks - i), 2, PAGE, n_kv, d).float()
            x[:, 0] *= gain
            c, sc = _codes(x, case["fmt"])
            s["codes"][i:i + step], s["scales"][i:i + step] = c, sc.permute(0, 3, 1, 2)
    if case["op"] == "decode":
        s["q"] = randn(len(lens), case["n_q"], d)
        return s
    packed, pages = _packed(lens)
    s["dst"] = i32(packed)
    s["pool"] = torch.zeros((pages, 2, PAGE, n_kv, d), device=_dev(), dtype=dt)
    return s


def _codes(x, fmt):
    """fp32 rows (..., d) -> codes and their scales (...)."""
    kind, top = _FMT[fmt]
    a = x.abs().amax(-1)
    a = torch.where(a < TINY, 0.0, a)
    y = x * torch.where(a > 0, top / a, 0.0).unsqueeze(-1)
    return (torch.round(y) if fmt == "int8" else y).to(kind), a / top


# ── one pass ─────────────────────────────────────────────────────────────────


def run(state):
    op = state["case"]["op"]
    if own:
        from vllm_mps_b200 import kernels as K

        if op == "decode":
            return K.paged_decode_attention_cache8(state["q"], K.KVCache8(state["codes"], state["scales"]),
                                                   state["bt"], state["lens"])
        if op == "read":
            return K.read_cache8(K.KVCache8(state["codes"], state["scales"]), state["bt"],
                                 state["lens"], state["pool"], state["dst"])
        case = state["case"]
        nq, nk = case["n_q"] * case["d"], case["n_kv"] * case["d"]
        qkv = state["qkv"]
        eight = case["fmt"] != "none"
        cache = K.KVCache8(state["codes"], state["scales"]) if eight else state["pool"]
        q = K.norm_rope_and_cache(qkv[:, :nq], qkv[:, nq:nq + nk], qkv[:, nq + nk:], state["positions"],
                                  state["slots"], state["inv_freq"], cache, state["q_weight"],
                                  state["k_weight"], EPS)
        if eight:
            K.read_cache8(cache, state["bt"], state["lens"], state["pool"], state["dst"])
        return dict(q=q, pool=state["pool"])
    return {"store": _plain_store, "read": _plain_read, "decode": _plain_decode}[op](state)


def _plain_rotate(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_store(s):
    case = s["case"]
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    q, k, v = s["qkv"].unflatten(1, (n_q + 2 * n_kv, d)).split([n_q, n_kv, n_kv], 1)
    angle = s["positions"].double().unsqueeze(1) * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    q = _plain_rotate(q, s["q_weight"], cos, sin).to(q.dtype)
    k = _plain_rotate(k, s["k_weight"], cos, sin)
    slot = s["slots"].long()
    blk, off = slot // PAGE, slot % PAGE
    if case["fmt"] == "none":
        s["pool"][blk, 0, off] = k.to(q.dtype)
        s["pool"][blk, 1, off] = v
        return dict(q=q, pool=s["pool"])
    for kind, x in ((0, k), (1, v.float())):
        c, sc = _codes(x, case["fmt"])
        # Indexed writes know no 8-bit floats: the same bytes as integers.
        s["codes"].view(torch.int8)[blk, kind, off] = c.view(torch.int8)
        s["scales"][blk, :, kind, off] = sc
    return dict(q=q, pool=_plain_read(s))


def _plain_read(s):
    n = s["lens"].long()
    pages = s["bt"].shape[1]
    t = torch.arange(pages * PAGE, device=n.device).view(pages, PAGE)
    live = t < n[:, None, None]
    b, i = live.any(2).nonzero(as_tuple=True)
    src, dst = s["bt"][b, i].long(), s["dst"][b, i].long()
    x = s["codes"].view(torch.int8)[src].view(s["codes"].dtype).float()
    x = x * s["scales"][src].permute(0, 2, 3, 1).unsqueeze(-1)
    s["pool"][dst] = torch.where(live[b, i][:, None, :, None, None], x, 0.0).to(s["pool"].dtype)
    return s["pool"]


def _plain_decode(s):
    q, bt = s["q"], s["bt"].long()
    B, P = bt.shape
    n_kv, d = s["codes"].shape[3:]
    G, L = q.shape[1] // n_kv, P * PAGE

    def values(kind):
        x = s["codes"].view(torch.int8)[:, kind][bt].view(s["codes"].dtype).float()
        x = x * s["scales"][:, :, kind][bt].transpose(2, 3).unsqueeze(-1)
        return x.reshape(B, L, n_kv, d).transpose(1, 2)

    x = torch.matmul(q.float().view(B, n_kv, G, d), values(0).transpose(2, 3)) * (1.0 / math.sqrt(d))
    live = torch.arange(L, device=q.device) < s["lens"].long()[:, None, None, None]
    x = torch.where(live, x, float("-inf"))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(e, values(1)) / e.sum(-1, keepdim=True)
    return o.reshape(q.shape).to(q.dtype)


# ── the same in 64 bits, from the definitions ────────────────────────────────


def _stored64(x, fmt):
    """What double rows (..., d) read back as."""
    top = 127.0 if fmt == "int8" else 448.0
    scale = x.abs().max(-1, keepdim=True).values / top
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale
    # e4m3: four significant bits, exponents from -6 up.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0) * scale


def exact(case, seed):
    s = prepare(case, seed)
    n_kv, d = case["n_kv"], case["d"]
    lens = _lens(case)
    if case["op"] == "store":
        n_q = case["n_q"]
        seq, pos = _rows(case, lens)
        x = s["qkv"].double().view(len(pos), n_q + 2 * n_kv, d)
        at = torch.tensor(pos, dtype=torch.float64, device=x.device)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                           torch.einsum("r,j->rj", at, s["inv_freq"].double()))
        parts = []
        for h0, h1, w in ((0, n_q, s["q_weight"]), (n_q, n_q + n_kv, s["k_weight"])):
            y = x[:, h0:h1]
            if w is not None:
                y = y * w.double() / torch.sqrt(y.square().sum(-1, keepdim=True) / d + EPS)
            z = torch.complex(y[..., : d // 2], y[..., d // 2:]) * turn.unsqueeze(1)
            parts.append(torch.cat([z.real, z.imag], -1))
        q, k = parts
        v = x[:, n_q + n_kv:]
        if case["fmt"] != "none":
            k, v = _stored64(k, case["fmt"]), _stored64(v, case["fmt"])
        pool = s["pool"].double()
        dst = s["bt"] if case["fmt"] == "none" else s["dst"]
        row = torch.tensor(pos, device=x.device)
        blk = dst[torch.tensor(seq, device=x.device), row // PAGE].long()
        pool[blk, 0, row % PAGE], pool[blk, 1, row % PAGE] = k, v
        return dict(q=q, pool=pool)
    if case["op"] == "read":
        pool = s["pool"].double()
        for i, n in enumerate(lens):
            for page in range(0, (n + PAGE - 1) // PAGE, 1024):
                ids = s["bt"][i, page:min(page + 1024, (n + PAGE - 1) // PAGE)].long().tolist()
                c = torch.stack([s["codes"][b] for b in ids]).double()
                sc = torch.stack([s["scales"][b] for b in ids]).double()
                x = torch.einsum("pktnd,pnkt->pktnd", c, sc)
                over = (page + len(ids)) * PAGE - n
                if over > 0:
                    x[-1, :, PAGE - over:] = 0
                pool[s["dst"][i, page:page + len(ids)].long()] = x
        return pool
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    G = case["n_q"] // n_kv
    wide = s["codes"].view(torch.uint8)
    for i, n in enumerate(lens):
        ids = s["bt"][i, : (n + PAGE - 1) // PAGE].long()
        kv = wide[ids].view(s["codes"].dtype)
        sc = s["scales"][ids].double()
        for h in range(n_kv):
            k = (kv[:, 0, :, h].double() * sc[:, h, 0].unsqueeze(-1)).flatten(0, 1)[:n]
            v = (kv[:, 1, :, h].double() * sc[:, h, 1].unsqueeze(-1)).flatten(0, 1)[:n]
            x = torch.einsum("gd,td->gt", s["q"][i, h * G:(h + 1) * G].double(), k) / math.sqrt(d)
            out[i, h * G:(h + 1) * G] = torch.einsum("gt,td->gd", torch.softmax(x, -1), v)
    return out


# ── what a pass cannot do without ────────────────────────────────────────────


def work(case):
    lens = _lens(case)
    n_kv, d = case["n_kv"], case["d"]
    side = 4 * sum((n + PAGE - 1) // PAGE for n in lens) + 4 * len(lens)
    eight, sixteen = 2 * n_kv * (d + 4), 4 * n_kv * d  # bytes of one token's K and V
    if case["op"] == "decode":
        n_q = case["n_q"]
        return dict(bytes=sum(lens) * eight + side + 4 * len(lens) * n_q * d,
                    flops=4 * n_q * d * sum(lens))
    if case["op"] == "read":
        return dict(bytes=sum(lens) * (eight + sixteen) + 2 * side, flops=2 * n_kv * d * sum(lens))
    rows = len(lens) if case["rows"] else sum(lens)
    heads = case["n_q"] + n_kv
    data = rows * (2 * (heads + n_kv) * d + 2 * case["n_q"] * d + 8)
    data += rows * sixteen if case["fmt"] == "none" else rows * (eight + sixteen) + 2 * side
    return dict(bytes=data, flops=rows * heads * d * (9 if case["norm"] else 3))
