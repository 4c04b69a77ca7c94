"""Cases that measure the operators of drafted (speculative) decoding over a paged cache.

One step of such a decoder: every sequence brings its current token and a tree
of drafted continuations, the attention runs over the cache and the tree, a
token is drawn after every node, and the longest path of drafts that the drawn
tokens agree with stays in the cache.  ``run`` computes the three operators in a
plain form (elementary torch operations in 32 bits, angles, probabilities and
their sums in 64), or through the library's entry points where ``own`` is true.

Trees are packed rows: ``cu_seqlens`` holds where each sequence's nodes start,
``kv_lens`` its length with them.  Node ``i`` of ``n`` lies in place
``kv_len - n + i`` of the cache and stands at position ``kv_len - n + depth``;
``parents`` holds the index of its parent among the sequence's nodes, or -1.
It sees what was in the cache before, its ancestors and itself; with a window
``W > 0`` of those only positions ``> p - W`` and the first ``sinks`` ones.

A token is drawn from ``softmax(logits / temperature)``, restricted in the order
of falling logits (equal ones by the lower id) to the first ``top_k``, of those
to the fewest that hold ``top_p`` of their sum, and to probabilities of at least
``min_p`` times the largest: the first id whose running sum, over kept ids in
rising order, exceeds ``uniform`` times the whole.  With it comes the logarithm of
its probability in the restricted distribution.
"""

from __future__ import annotations

import math
import random

import torch

own = False

HD = 128
THETA = 1e6
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one step of the decoder stack's generation with small trees: batch 8 after prompts of 512 (latency)
        dict(name="tree 8 x 8 over 512-639", op="tree", seqs=8, lo=512, hi=639, nlo=8, nhi=8, nq=32, nkv=4, page=16,
             window=0, sinks=0),
        # one user with a long text
        dict(name="tree 1 x 13 over 30011", op="tree", seqs=1, lo=30011, hi=30011, nlo=13, nhi=13, nq=32, nkv=4,
             page=64, window=0, sinks=0),
        # a server's step over sequences of every age
        dict(name="tree 40 ragged", op="tree", seqs=40, lo=1, hi=32768, nlo=3, nhi=16, nq=32, nkv=4, page=64, window=0,
             sinks=0),
        # the widest trees, more rows than one tile, long streams in a window with four first tokens
        dict(name="tree 16 x 49-64 window", op="tree", seqs=16, lo=1500, hi=30011, nlo=49, nhi=64, nq=32, nkv=4,
             page=32, window=4096, sinks=4),
        # a generation step's draw: batch 8, the usual filters
        dict(name="sample 8 top-k top-p", op="sample", rows=8, vocab=151936, f32=False, temperature=0.6, top_k=20,
             top_p=0.95, min_p=0.0, mixed=False, masked=0.0),
        # three rows in fp32 from everything
        dict(name="sample 3 f32", op="sample", rows=3, vocab=151936, f32=True, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, mixed=False, masked=0.0),
        # a server's batch: each request with its own settings, some greedy, some with tokens masked out
        dict(name="sample 100 mixed", op="sample", rows=100, vocab=151936, f32=False, temperature=1.0, top_k=50,
             top_p=0.9, min_p=0.05, mixed=True, masked=0.3),
        # the nodes of 64 trees of 16, top-p alone
        dict(name="sample 1024 top-p", op="sample", rows=1024, vocab=151936, f32=False, temperature=0.8, top_k=0,
             top_p=0.9, min_p=0.0, mixed=False, masked=0.0),
        # fp32 logits, an odd vocabulary, min-p alone
        dict(name="sample 257 f32 min-p", op="sample", rows=257, vocab=50257, f32=True, temperature=1.3, top_k=0,
             top_p=1.0, min_p=0.05, mixed=False, masked=0.0),
        # the accepted paths of the first case's trees, keys and values of 48 layers
        dict(name="accept 8 x 8", op="accept", seqs=8, nodes=8, deep=4, past=520, planes=96, nkv=4, page=16),
        # a server's step, larger trees
        dict(name="accept 64 x 31", op="accept", seqs=64, nodes=31, deep=8, past=41, planes=96, nkv=4, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "sample", "sample", "sample", "accept"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "tree":
        nq, nkv = rng.choice([(32, 4), (32, 4), (32, 8), (16, 2), (8, 8), (16, 1), (12, 4), (40, 8), (28, 4)])
        window, sinks = (_log(rng, 1, 8000), rng.choice([0, 1, 4, 17, 128])) if rng.random() < 0.4 else (0, 0)
        seqs, nhi = _log(rng, 1, 48), _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, min(65536, 600000 // (seqs * nkv), 300_000_000 // (seqs * nq * nhi))))
        return dict(op=op, seqs=seqs, lo=_log(rng, 1, hi), hi=hi, nlo=_log(rng, 1, nhi), nhi=nhi, nq=nq, nkv=nkv,
                    page=page, window=window, sinks=sinks)
    if op == "sample":
        vocab = _log(rng, 100, 160000)
        rows = _log(rng, 1, min(2048, 150_000_000 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, f32=rng.random() < 0.4, temperature=rng.choice([0.3, 0.7, 1.0, 1.5]),
                    top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), mixed=rng.random() < 0.3,
                    masked=rng.choice([0.0, 0.0, 0.5]))
    seqs, nodes, nkv, planes = _log(rng, 1, 64), _log(rng, 3, 64), rng.choice([1, 2, 4, 8]), 2 * _log(rng, 1, 48)
    most = 3_000_000_000 // (seqs * planes * nkv * HD * 2)  # positions of a sequence that the pool holds at most
    past = _log(rng, 1, max(1, min(600, most - nodes - page)))
    return dict(op=op, seqs=seqs, nodes=nodes, deep=_log(rng, 1, min(12, nodes - 1)), past=past, planes=planes, nkv=nkv,
                page=page)


def _between(lo, hi, n):
    """n whole numbers even over the logarithm from lo to hi."""
    return [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * (i / (n - 1) if n > 1 else 1))) for i in range(n)]


def _lengths(case):
    """What each sequence of a tree case holds already, and its nodes (long ones and large trees mixed)."""
    nodes = _between(case["nlo"], case["nhi"], case["seqs"])
    random.Random(case["seqs"]).shuffle(nodes)
    return _between(case["lo"], case["hi"], case["seqs"]), nodes


def _depths(case):
    """How many nodes of each tree are accepted."""
    return [1 + i % case["deep"] for i in range(case["seqs"])]


def work(case):
    op = case["op"]
    if op == "sample":
        n, size = case["rows"] * case["vocab"], 4 if case["f32"] else 2
        return {"bytes": n * size + case["rows"] * (12 + (20 if case["mixed"] else 4)), "flops": 5 * n}
    if op == "accept":
        moved = sum(d - 1 for d in _depths(case))
        return {"bytes": 2 * moved * case["planes"] * case["nkv"] * HD * 2 + case["seqs"] * case["nodes"] * (8 + 8 + 4 + 12),
                "flops": 0}
    nq, nkv, w, sinks = case["nq"], case["nkv"], case["window"], case["sinks"]
    pasts, nodes = _lengths(case)
    rows = sum(nodes)
    held = [n if not w else min(n, w - 1) + min(sinks, max(0, n - w + 1)) for n in pasts]  # what a tree's root sees
    return {"bytes": 2 * HD * (2 * nkv * sum(held) + rows * (nq + 2 * nkv + 2 * nkv + nq)),
            "flops": 4 * HD * nq * sum(n * (h + 1) for n, h in zip(nodes, held))}


# ------------------------------------------------------------------ inputs
def _pages(case, total, host):
    """Page ids of sequences of these lengths, anywhere in a pool, and the pool's size."""
    ps = case["page"]
    need = (total + ps - 1) // ps
    held = int(need.sum())
    pool = held + max(1, held // 16)
    table = torch.full((len(total), int(need.max())), -1, dtype=torch.int32)
    table[torch.arange(table.shape[1])[None] < need[:, None]] = torch.randperm(pool, generator=host)[:held].to(torch.int32)
    return table, pool


def _starts(counts):
    cu = torch.zeros(len(counts) + 1, dtype=torch.int32)
    cu[1:] = counts.cumsum(0)
    return cu


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0, shift=0.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(shift, scale, generator=g)

    op = case["op"]
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad bulk and a few tokens that stand out of it
        logits = normal(rows, vocab, dtype=torch.float32, scale=2.0)
        at = torch.randint(vocab, (rows, 48), generator=g, device=dev)
        logits.scatter_add_(1, at, 9 * torch.rand(rows, 48, generator=g, device=dev))
        if case["masked"]:
            logits[torch.rand(rows, vocab, generator=g, device=dev) < case["masked"]] = -math.inf
        state = {"case": case, "logits": logits if case["f32"] else logits.bfloat16(),
                 "uniforms": torch.rand(rows, generator=g, device=dev)}
        for name, default, others in (("temperature", case["temperature"], [0.0, 0.5, 1.0]), ("top_k", case["top_k"], [0, 5]),
                                      ("top_p", case["top_p"], [1.0, 0.8]), ("min_p", case["min_p"], [0.0, 0.2])):
            state[name] = default
            if case["mixed"]:  # each row its own
                choice = torch.tensor([default] + others, dtype=torch.int32 if name == "top_k" else torch.float32)
                state[name] = choice[torch.randint(len(choice), (rows,), generator=host)].to(dev)
        return state
    if op == "accept":
        n, b = case["nodes"], case["seqs"]
        tokens = torch.randint(1000, (b, n), generator=host)
        sampled = torch.randint(1000, 2000, (b, n), generator=host)
        parents = torch.empty(b, n, dtype=torch.int32)
        for q, deep in enumerate(_depths(case)):
            parents[q] = torch.tensor([-1] + [int(torch.randint(i, (1,), generator=host)) for i in range(1, n)])
            # one path is agreed with; the first draft is never on it, so every node of it has to move
            path = [0] + sorted((torch.randperm(n - 2, generator=host)[:deep - 1] + 2).tolist())
            for a, c in zip(path, path[1:]):
                parents[q, c], sampled[q, a] = a, tokens[q, c]
                for i in range(a + 1, c):
                    tokens[q, i] += 5000 * int(parents[q, i] == a)
        counts = torch.full((b,), n)
        total = counts + case["past"]
        table, pool = _pages(case, total, host)
        return {"case": case, "tokens": tokens.reshape(-1).to(dev), "sampled": sampled.reshape(-1).to(dev),
                "parents": parents.reshape(-1).to(dev), "cu_seqlens": _starts(counts).to(dev),
                "kv_lens": total.to(torch.int32).to(dev), "page_table": table.to(dev),
                "pages": normal(case["planes"], pool, case["nkv"], case["page"], HD)}

    nq, nkv, b = case["nq"], case["nkv"], case["seqs"]
    order = torch.randperm(b, generator=host)
    past, counts = (torch.tensor(x)[order] for x in _lengths(case))
    total = past + counts
    table, pool = _pages(case, total, host)
    parents = []
    for n in counts.tolist():  # half of the nodes continue the one before them
        parents += [-1] + [i - 1 if torch.rand(1, generator=host) < 0.5 else int(torch.randint(i, (1,), generator=host))
                           for i in range(1, n)]
    rows = int(counts.sum())
    return {"case": case, "k_pages": normal(pool, nkv, case["page"], HD), "v_pages": normal(pool, nkv, case["page"], HD),
            "page_table": table.to(dev), "parents": torch.tensor(parents, dtype=torch.int32).to(dev),
            "cu_seqlens": _starts(counts).to(dev), "kv_lens": total.to(torch.int32).to(dev),
            "longest": int(counts.max()), "qkv": normal(rows, (nq + 2 * nkv) * HD),
            "q_weight": normal(HD, scale=0.2, shift=1.2), "k_weight": normal(HD, scale=0.2, shift=1.0)}


# ------------------------------------------------------------------ one pass
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _own_tree(s):
    from nki_moe_b200 import ops
    c = s["case"]
    out = ops.paged_tree_attention(s["qkv"], s["q_weight"], s["k_weight"], s["parents"], s["cu_seqlens"], s["kv_lens"],
                                   s["k_pages"], s["v_pages"], s["page_table"], c["nq"], c["nkv"], theta=THETA, eps=EPS,
                                   window=c["window"], sinks=c["sinks"])
    return out, s["k_pages"], s["v_pages"]


def _own_sample(s):
    from nki_moe_b200 import ops
    return tuple(ops.sample_tokens(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"]))


def _own_accept(s):
    from nki_moe_b200 import ops
    counts, path, new = ops.accept_drafts(s["tokens"], s["sampled"], s["parents"], s["cu_seqlens"], s["kv_lens"],
                                          s["pages"], s["page_table"])
    return counts, path, new, s["pages"]


# ------------------------------------------------------------------ plain forms
def _norm_rope(x, weight, positions):
    """RMSNorm over each head of x [rows, heads, 128] and rotate-half positions, in 32 bits; the angles in 64."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    freq = THETA ** (-torch.arange(HD // 2, dtype=torch.float64, device=x.device) / (HD // 2))
    angle = positions.double()[:, None, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = x[..., :HD // 2], x[..., HD // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_tree(s):
    c = s["case"]
    nq, nkv, w, sinks = c["nq"], c["nkv"], c["window"], c["sinks"]
    table, cu, kv, parents = s["page_table"], s["cu_seqlens"].long(), s["kv_lens"].long(), s["parents"].long()
    b, rows, longest, dev = table.shape[0], s["qkv"].shape[0], s["longest"], s["qkv"].device
    counts = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(b, device=dev), counts, output_size=rows)
    at = torch.arange(rows, device=dev) - cu[seq]
    past = (kv - counts)[seq]
    # up the trees, one generation at a time
    line = torch.zeros(rows, longest, dtype=torch.bool, device=dev)  # of each row: itself and its ancestors
    line[torch.arange(rows, device=dev), at] = True
    depth, cur = torch.zeros_like(at), parents
    for _ in range(longest - 1):
        up = cur >= 0
        depth += up
        line |= (torch.arange(longest, device=dev) == cur[:, None]) & up[:, None]
        cur = torch.where(up, parents[cu[seq] + cur.clamp(min=0)], cur)
    pos, place = past + depth, past + at
    heads = s["qkv"].view(rows, nq + 2 * nkv, HD)
    q = _norm_rope(heads[:, :nq], s["q_weight"], pos)
    ps = c["page"]
    page, row = table[seq, place // ps].long(), place % ps
    s["k_pages"][page, :, row] = _norm_rope(heads[:, nq:nq + nkv], s["k_weight"], pos).to(torch.bfloat16)
    s["v_pages"][page, :, row] = heads[:, nq + nkv:]
    keys, values = (x[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, HD).float()
                    for x in (s["k_pages"], s["v_pages"]))
    # the position that stands in each place, for each row -1 where it is not of its line or of before
    n_keys = keys.shape[2]
    k = torch.arange(n_keys + longest, device=dev)
    where = torch.where(k < past[:, None], k, -1)
    in_tree = torch.zeros(b, longest, dtype=torch.long, device=dev)
    in_tree[seq, at] = pos
    where.scatter_(1, past[:, None] + k[:longest], torch.where(line, in_tree[seq], -1))
    where = where[:, :n_keys]
    seen = where >= 0
    if w:
        seen &= (where > pos[:, None] - w) | (where < sinks)
    qs = torch.zeros(b, longest, nq, HD, device=dev)
    qs[seq, at] = q
    mask = torch.zeros(b, longest, n_keys, dtype=torch.bool, device=dev)
    mask[..., 0] = True  # rows that only pad see the first place
    mask[seq, at] = seen
    grp = nq // nkv
    qs = qs.view(b, longest, nkv, grp, HD).permute(0, 2, 3, 1, 4).reshape(b, nkv, grp * longest, HD)
    sc = torch.matmul(qs, keys.transpose(-1, -2)).mul_(HD ** -0.5)
    sc.view(b, nkv, grp, longest, n_keys).masked_fill_(~mask[:, None, None], -math.inf)
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    o = (torch.matmul(sc, values) / sc.sum(-1, keepdim=True)).view(b, nkv, grp, longest, HD)
    out = o.permute(0, 3, 1, 2, 4).reshape(b, longest, nq * HD)[seq, at].to(torch.bfloat16)
    return out, s["k_pages"], s["v_pages"]


def _column(value, rows, dev, dtype):
    """A setting as one column."""
    if not isinstance(value, torch.Tensor):
        value = torch.full((rows,), value, dtype=dtype, device=dev)
    return value.to(dtype)[:, None]


def _plain_sample(s):
    rows, vocab = s["logits"].shape
    dev, u = s["logits"].device, s["uniforms"].double()[:, None]
    t, p, m = (_column(s[x], rows, dev, torch.float64) for x in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], rows, dev, torch.int64)
    parts = []
    for r in range(0, rows, 64):  # so many rows at a time as memory likes
        e = slice(r, r + 64)
        x, ids = torch.sort(s["logits"][e].float(), dim=-1, descending=True, stable=True)
        d = x.double() - x[:, :1].double()
        wt = (d / torch.where(t[e] > 0, t[e], 1.0)).exp()
        place = torch.arange(vocab, device=dev)
        keep = (place < torch.where(k[e] > 0, k[e], vocab)) & (wt >= m[e])
        wt_k = torch.where((place < torch.where(k[e] > 0, k[e], vocab)), wt, 0.0)
        run_to = wt_k.cumsum(-1)
        keep &= (run_to - wt_k < p[e] * run_to[:, -1:]) | (p[e] >= 1)
        keep &= (t[e] > 0) | (place == 0)
        keep[:, 0] = True
        kept = torch.zeros_like(wt).scatter_(1, ids, torch.where(keep, wt, 0.0))
        total = kept.cumsum(-1)
        over = (total > u[e] * total[:, -1:]) & (kept > 0)
        drawn = over.to(torch.int8).argmax(-1, keepdim=True)
        parts.append((drawn[:, 0], (kept.gather(-1, drawn) / total[:, -1:]).log()[:, 0].float()))
    return tuple(torch.cat(x) for x in zip(*parts))


def _plain_accept(s):
    c = s["case"]
    b, n, ps = c["seqs"], c["nodes"], c["page"]
    tok, sam, par = (s[x].view(b, n).long() for x in ("tokens", "sampled", "parents"))
    dev = tok.device
    cur = torch.zeros(b, dtype=torch.long, device=dev)
    alive = torch.ones(b, dtype=torch.bool, device=dev)
    path = torch.full((b, n), -1, dtype=torch.long, device=dev)
    path[:, 0] = 0
    for i in range(1, n):
        fits = (par == cur[:, None]) & (tok == sam.gather(1, cur[:, None])) & alive[:, None]
        fits &= torch.arange(n, device=dev) > cur[:, None]
        alive = fits.any(-1)
        cur = torch.where(alive, fits.to(torch.int8).argmax(-1), cur)
        path[:, i] = torch.where(alive, cur, torch.full_like(cur, -1))
    on = path >= 0
    counts = on.sum(-1)
    new = torch.where(on, sam.gather(1, path.clamp(min=0)), torch.full_like(sam, -1))
    past = s["kv_lens"].long()[:, None] - n
    seq = torch.arange(b, device=dev)[:, None]
    # nodes that stay in no place are copied onto themselves
    own_place = torch.arange(n, device=dev).expand(b, n)
    src, dst = past + torch.where(on, path, own_place), past + own_place
    got = s["pages"][:, s["page_table"][seq, src // ps].long(), :, src % ps]
    s["pages"][:, s["page_table"][seq, dst // ps].long(), :, dst % ps] = got
    return counts.to(torch.int32), path.to(torch.int32).view(-1), new.view(-1), s["pages"]


_OWN = {"tree": _own_tree, "sample": _own_sample, "accept": _own_accept}
_PLAIN = {"tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept}


# ------------------------------------------------------------------ in 64 bits
def _turn(head, weight, p):
    """One sequence's heads [rows, heads, 128] at positions p, normed and turned as complex numbers."""
    head = head.double()
    head = head / ((head ** 2).sum(-1, keepdim=True) / HD + EPS).sqrt() * weight.double()
    z = torch.complex(head[..., :HD // 2], head[..., HD // 2:])
    i = torch.arange(HD // 2, dtype=torch.float64, device=head.device)
    by = p.double()[:, None] / torch.exp(i / (HD // 2) * math.log(THETA))
    z = z * torch.polar(torch.ones_like(by), by)[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_tree(case, s):
    nq, nkv, ps = case["nq"], case["nkv"], case["page"]
    cu, total, table = s["cu_seqlens"].tolist(), s["kv_lens"].tolist(), s["page_table"].tolist()
    parents, outs = s["parents"].tolist(), []
    for b in range(case["seqs"]):
        n = cu[b + 1] - cu[b]
        past, up = total[b] - n, parents[cu[b]:cu[b + 1]]
        lines = []  # each node's path from the root
        for i in range(n):
            lines.append((lines[up[i]] if up[i] >= 0 else []) + [i])
        p = torch.tensor([past + len(x) - 1 for x in lines], device="cuda")
        place = torch.arange(past, total[b], device="cuda")
        pages = torch.tensor([x for x in table[b] if x >= 0], device="cuda")
        heads = s["qkv"][cu[b]:cu[b + 1]].view(n, nq + 2 * nkv, HD)
        q = _turn(heads[:, :nq], s["q_weight"], p)
        # the cache holds the new keys in its own type
        new = _turn(heads[:, nq:nq + nkv], s["k_weight"], p).to(torch.bfloat16)
        for j in range(nkv):
            s["k_pages"][pages[place // ps], j, place % ps] = new[:, j]
            s["v_pages"][pages[place // ps], j, place % ps] = heads[:, nq + nkv + j]
        k, v = (s[x][pages].transpose(0, 1).reshape(nkv, -1, HD)[:, :total[b]].double() for x in ("k_pages", "v_pages"))
        hidden = torch.ones(n, total[b], dtype=torch.bool, device="cuda")
        at = torch.arange(past, device="cuda")
        for i, x in enumerate(lines):
            here = past + len(x) - 1
            hidden[i, :past] = (at <= here - case["window"]) & (at >= case["sinks"]) if case["window"] else False
            for d, a in enumerate(x):
                out = case["window"] and past + d <= here - case["window"] and past + d >= case["sinks"]
                hidden[i, past + a] = bool(out)
        o = torch.empty_like(q)
        for h in range(nq):
            wt = q[:, h] @ k[h * nkv // nq].T / math.sqrt(HD)
            wt[hidden] = -math.inf
            o[:, h] = torch.softmax(wt, -1) @ v[h * nkv // nq]
        outs.append(o.reshape(n, nq * HD))
    return torch.cat(outs), s["k_pages"], s["v_pages"]


def _exact_sample(case, s):
    def of(name, i):
        return float(s[name][i]) if isinstance(s[name], torch.Tensor) else s[name]

    out, logs = [], []
    for i in range(case["rows"]):
        x = s["logits"][i].double()
        t, k = of("temperature", i), int(of("top_k", i))
        if t == 0:
            out.append(int((x == x.max()).nonzero()[0]))
            logs.append(0.0)
            continue
        ids = torch.argsort(x, descending=True, stable=True)
        if k > 0:
            ids = ids[:k]
        x = x[ids] / t
        prob = torch.softmax(x, 0)
        least = of("min_p", i) * prob[0]
        if of("top_p", i) < 1:
            n = int(torch.searchsorted(prob.cumsum(0), of("top_p", i))) + 1
            ids, prob, x = ids[:n], prob[:n], x[:n]
        ids, x, prob = ids[prob >= least], x[prob >= least], prob[prob >= least]
        ids, order = torch.sort(ids)
        upto = prob[order].cumsum(0)
        at = int(torch.searchsorted(upto, float(s["uniforms"][i]) * upto[-1], right=True))
        at = min(at, len(ids) - 1)
        out.append(int(ids[at]))
        logs.append(float(x[order[at]] - torch.logsumexp(x, 0)))
    return torch.tensor(out, device="cuda"), torch.tensor(logs, dtype=torch.float64, device="cuda")


def _exact_accept(case, s):
    n, ps = case["nodes"], case["page"]
    tok, sam, par = (s[x].view(-1, n).tolist() for x in ("tokens", "sampled", "parents"))
    table, lens = s["page_table"].tolist(), s["kv_lens"].tolist()
    counts, paths, news, pages = [], [], [], s["pages"].clone()
    for b in range(case["seqs"]):
        path = [0]
        while True:
            nxt = [i for i in range(path[-1] + 1, n) if par[b][i] == path[-1] and tok[b][i] == sam[b][path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        for to, a in enumerate(path):
            f, d = lens[b] - n + a, lens[b] - n + to
            pages[:, table[b][d // ps], :, d % ps] = s["pages"][:, table[b][f // ps], :, f % ps]
        counts.append(len(path))
        paths += path + [-1] * (n - len(path))
        news += [sam[b][i] for i in path] + [-1] * (n - len(path))
    dev = pages.device
    return (torch.tensor(counts, dtype=torch.int32, device=dev), torch.tensor(paths, dtype=torch.int32, device=dev),
            torch.tensor(news, device=dev), pages)


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "sample": _exact_sample, "accept": _exact_accept}[case["op"]](case, s)
