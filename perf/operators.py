"""Cases that measure the operators of serving with a paged key-value cache.

Five operators of one serving path: the store of a prompt's keys and values in
the pages of a cache, the prompt's attention over those pages, the attention of
one new token over them, the copies that fork and compact pages, and the log
probabilities of the tokens that come out.  ``run`` computes them in a plain
form (elementary torch operations in 32 bits, angles in 64), or through the
library's entry points where ``own`` is true.

The cache of a layer is ``k_pages`` / ``v_pages`` ``[pages, kv heads, page
size, 128]`` bf16; row ``b`` of ``page_table`` lists the pages of sequence
``b`` in order (-1: not held).  Prompts are packed rows: ``cu_seqlens`` holds
where each sequence's new rows start, ``kv_lens`` its length with them, so row
``i`` of ``n`` new ones stands at position ``kv_len - n + i``.  With a window
``W > 0`` the query at position ``p`` sees the keys ``p - W < s <= p`` and the
first ``sinks`` ones.
"""

from __future__ import annotations

import math

import torch

own = False

HD = 128
THETA = 1e6
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one step of the decoder stack's generation: batch 8, 128 tokens after prompts of 512 (latency)
        dict(name="decode 8 x 512-639", op="decode", seqs=8, lo=512, hi=639, nq=32, nkv=4, page=16, window=0, sinks=0),
        # a server's step over sequences of every age: one token to 32768
        dict(name="decode 48 ragged", op="decode", seqs=48, lo=1, hi=32768, nq=32, nkv=4, page=64, window=0, sinks=0),
        # long streams kept in a window with four first tokens, odd lengths
        dict(name="decode 24 window", op="decode", seqs=24, lo=1500, hi=30011, nq=32, nkv=4, page=32, window=2048,
             sinks=4),
        # the decoder stack's prompts: 8 x 512 tokens
        dict(name="prompt 8 x 512", op="prefill", seqs=8, lo=512, hi=512, past=0, nq=32, nkv=4, page=16, window=0,
             sinks=0),
        # one long prompt
        dict(name="prompt 8192", op="prefill", seqs=1, lo=8192, hi=8192, past=0, nq=32, nkv=4, page=64, window=0,
             sinks=0),
        # odd chunks of long prompts over what the cache holds of them, window and first tokens
        dict(name="chunk 4 window", op="prefill", seqs=4, lo=61, hi=509, past=9001, nq=32, nkv=4, page=64, window=4096,
             sinks=4),
        # the store of a few tokens of three sequences (latency)
        dict(name="store 3 x 1-7", op="store", seqs=3, lo=1, hi=7, past=100, nq=32, nkv=4, page=16),
        # the store of a prefill batch: 4 prompts around 2048 tokens
        dict(name="store 4 x 2001-2095", op="store", seqs=4, lo=2001, hi=2095, past=0, nq=32, nkv=4, page=64),
        # eight sequences forked: the last page of each, in the key and value pools of 48 layers
        dict(name="fork 8", op="copy", pairs=8, planes=96, nkv=4, page=16, pool=256),
        # a pool of 24 layers compacted
        dict(name="compact 300", op="copy", pairs=300, planes=48, nkv=4, page=64, pool=640),
        # a generation step's answer: batch 8, twenty alternatives
        dict(name="logprobs 8 top 20", op="logprobs", rows=8, vocab=151936, top=20, f32=False),
        # a prompt scored
        dict(name="logprobs 2000 top 5", op="logprobs", rows=2000, vocab=151936, top=5, f32=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "store", "copy", "logprobs"])
    nq, nkv = rng.choice([(32, 4), (32, 4), (32, 8), (16, 2), (8, 8), (16, 1), (12, 4), (40, 8), (28, 4)])
    page = rng.choice([16, 32, 64, 128, 256])
    window, sinks = (_log(rng, 1, 8000), rng.choice([0, 1, 4, 17, 128])) if rng.random() < 0.4 else (0, 0)
    if op == "decode":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, min(65536, 600000 // (seqs * nkv)))
        return dict(op=op, seqs=seqs, lo=_log(rng, 1, hi), hi=hi, nq=nq, nkv=nkv, page=page, window=window, sinks=sinks)
    if op == "prefill":
        seqs = _log(rng, 1, 16)
        hi = _log(rng, 1, min(4096, 16000 // seqs))
        past = rng.choice([0, 0, _log(rng, 1, 12000)])
        past = min(past, max(0, 25_000_000 // (seqs * hi) - hi))
        return dict(op=op, seqs=seqs, lo=_log(rng, 1, hi), hi=hi, past=past, nq=nq, nkv=nkv, page=page, window=window,
                    sinks=sinks)
    if op == "store":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 12000 // seqs)
        return dict(op=op, seqs=seqs, lo=_log(rng, 1, hi), hi=hi, past=rng.choice([0, _log(rng, 1, 30000)]), nq=nq,
                    nkv=nkv, page=page)
    if op == "copy":
        planes = 2 * _log(rng, 1, 48)
        most = 940_000_000 // (planes * nkv * page * HD * 2)
        pairs = _log(rng, 1, max(1, min(3000, most)))
        return dict(op=op, pairs=pairs, planes=planes, nkv=nkv, page=page, pool=2 * pairs + rng.randrange(1, 30))
    f32 = rng.random() < 0.4
    vocab = _log(rng, 100, 160000)
    rows = _log(rng, 1, min(8192, 150_000_000 // vocab))
    return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 32]), f32=f32)


def _spread(case):
    """The lengths of a case's sequences: even over the logarithm from lo to hi."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * (i / (n - 1) if n > 1 else 1))) for i in range(n)]


def _seen(case, p):
    """How many keys the query at position p sees."""
    w, s = case["window"], case["sinks"]
    return p + 1 if not w else min(p + 1, w) + min(s, max(0, p + 1 - w))


def work(case):
    op = case["op"]
    if op == "copy":
        return {"bytes": 2 * case["pairs"] * case["planes"] * case["nkv"] * case["page"] * HD * 2, "flops": 0}
    if op == "logprobs":
        n, size = case["rows"] * case["vocab"], 4 if case["f32"] else 2
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    nq, nkv, lens = case["nq"], case["nkv"], _spread(case)
    if op == "decode":
        seen = [_seen(case, n - 1) for n in lens]
        held = sum(seen) - len(seen)  # each sequence's new row comes with the step, not from the cache
        return {"bytes": 2 * HD * (2 * nkv * held + len(lens) * (nq + 2 * nkv + 2 * nkv + nq)),
                "flops": 4 * HD * nq * sum(seen)}
    rows = sum(lens)
    if op == "store":
        return {"bytes": 2 * HD * 2 * rows * (nq + 2 * nkv), "flops": 10 * HD * rows * (nq + nkv)}
    pairs = sum(_seen(case, case["past"] + i) for n in lens for i in range(n))
    keys = 0
    for n in lens:
        w, total = case["window"], case["past"] + n
        first = max(0, case["past"] - w + 1) if w else 0
        keys += total - first + min(case["sinks"], first)
    return {"bytes": 2 * HD * (2 * nkv * keys + 2 * nq * rows), "flops": 4 * HD * nq * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0, shift=0.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(shift, scale, generator=g)

    op = case["op"]
    if op == "copy":
        # pages in use anywhere in the pool go to free ones
        pages = normal(case["planes"], case["pool"], case["nkv"], case["page"], HD)
        at = torch.randperm(case["pool"], generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        n = case["pairs"]
        return {"case": case, "pages": pages, "src": at[:n].clone(), "dst": at[n:2 * n].clone()}
    if op == "logprobs":
        logits = normal(case["rows"], case["vocab"], dtype=torch.float32 if case["f32"] else torch.bfloat16, scale=2.5)
        tokens = torch.randint(case["vocab"], (case["rows"],), generator=g, device=dev)
        # most given tokens are likely ones
        tokens = torch.where(torch.rand(case["rows"], generator=g, device=dev) < 0.7, logits.argmax(-1), tokens)
        return {"case": case, "logits": logits, "tokens": tokens}

    nq, nkv, ps = case["nq"], case["nkv"], case["page"]
    host = torch.Generator().manual_seed(seed)
    lens = torch.tensor(_spread(case))[torch.randperm(case["seqs"], generator=host)]
    past = torch.zeros_like(lens) if op == "decode" else torch.full_like(lens, case["past"])
    total = lens + past
    need = (total + ps - 1) // ps
    held = int(need.sum())
    pool = held + max(1, held // 16)
    ids = torch.randperm(pool, generator=host)[:held].to(torch.int32)
    width = int(need.max())
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    table[torch.arange(width)[None] < need[:, None]] = ids
    state = {"case": case, "k_pages": normal(pool, nkv, ps, HD), "v_pages": normal(pool, nkv, ps, HD),
             "page_table": table.to(dev), "widest": int(total.max()), "longest": int(lens.max())}
    if op == "decode":
        state["positions"] = (total - 1).to(dev)
    else:
        cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
        cu[1:] = lens.cumsum(0)
        state["cu_seqlens"], state["kv_lens"] = cu.to(dev), total.to(torch.int32).to(dev)
    rows = len(lens) if op == "decode" else int(lens.sum())
    if op == "prefill":
        state["q"] = normal(rows, nq, HD, scale=1.3)
    else:
        state["qkv"] = normal(rows, (nq + 2 * nkv) * HD)
        state["q_weight"] = normal(HD, scale=0.2, shift=1.2)
        state["k_weight"] = normal(HD, scale=0.2, shift=1.0)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _own_decode(s):
    from nki_moe_b200 import ops
    c = s["case"]
    out = ops.paged_decode_attention(s["qkv"], s["q_weight"], s["k_weight"], s["positions"], s["k_pages"],
                                     s["v_pages"], s["page_table"], c["nq"], c["nkv"], theta=THETA, eps=EPS,
                                     window=c["window"], sinks=c["sinks"])
    return out, s["k_pages"], s["v_pages"]


def _own_prefill(s):
    from nki_moe_b200 import ops
    c = s["case"]
    return ops.paged_prefill_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_seqlens"],
                                       s["kv_lens"], window=c["window"], sinks=c["sinks"])


def _own_store(s):
    from nki_moe_b200 import ops
    c = s["case"]
    q = ops.qk_norm_rope_store(s["qkv"], s["q_weight"], s["k_weight"], s["cu_seqlens"], s["kv_lens"], s["k_pages"],
                               s["v_pages"], s["page_table"], c["nq"], c["nkv"], theta=THETA, eps=EPS)
    return q, s["k_pages"], s["v_pages"]


def _own_copy(s):
    from nki_moe_b200 import ops
    return ops.copy_pages(s["pages"], s["src"], s["dst"])


def _own_logprobs(s):
    from nki_moe_b200 import ops
    return tuple(ops.token_logprobs(s["logits"], s["tokens"], s["case"]["top"]))


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


def _put(pages, table, seq, pos, rows):
    ps = pages.shape[2]
    pages[table[seq, pos // ps].long(), :, pos % ps] = rows


def _held(pages, table):
    """The cache of each sequence as one [sequences, kv heads, positions, 128] tensor in 32 bits."""
    got = pages[table.clamp(min=0).long()]
    return got.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pages.shape[1], -1, HD).float()


def _sees(pos, keys, window, sinks):
    s = torch.arange(keys, device=pos.device)
    see = s <= pos[..., None]
    return see & ((s > pos[..., None] - window) | (s < sinks)) if window else see


def _attend(q, k, v, see):
    """q [b, kv heads, group, rows, 128], k and v [b, kv heads, keys, 128], see [b, rows, keys]."""
    s = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(HD ** -0.5)
    s.masked_fill_(~see[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    return torch.matmul(s, v[:, :, None]) / s.sum(-1, keepdim=True)


def _plain_decode(s):
    c = s["case"]
    nq, nkv, b = c["nq"], c["nkv"], s["qkv"].shape[0]
    pos, rows = s["positions"], s["qkv"].view(b, nq + 2 * nkv, HD)
    q = _norm_rope(rows[:, :nq], s["q_weight"], pos)
    k = _norm_rope(rows[:, nq:nq + nkv], s["k_weight"], pos)
    seq = torch.arange(b, device=pos.device)
    _put(s["k_pages"], s["page_table"], seq, pos, k.to(torch.bfloat16))
    _put(s["v_pages"], s["page_table"], seq, pos, rows[:, nq + nkv:])
    keys, values = _held(s["k_pages"], s["page_table"]), _held(s["v_pages"], s["page_table"])
    see = _sees(pos[:, None], keys.shape[2], c["window"], c["sinks"])
    o = _attend(q.view(b, nkv, nq // nkv, 1, HD), keys, values, see)
    return o.reshape(b, nq * HD).to(torch.bfloat16), s["k_pages"], s["v_pages"]


def _places(s):
    """Sequence, place among its new rows and position of each packed row."""
    cu, kv = s["cu_seqlens"].long(), s["kv_lens"].long()
    n = cu[1:] - cu[:-1]
    rows = s["q"].shape[0] if "q" in s else s["qkv"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(n), device=cu.device), n, output_size=rows)
    at = torch.arange(rows, device=cu.device) - cu[seq]
    return seq, at, (kv - n)[seq] + at


def _plain_store(s):
    c = s["case"]
    nq, nkv = c["nq"], c["nkv"]
    seq, _, pos = _places(s)
    rows = s["qkv"].view(-1, nq + 2 * nkv, HD)
    k = _norm_rope(rows[:, nq:nq + nkv], s["k_weight"], pos)
    _put(s["k_pages"], s["page_table"], seq, pos, k.to(torch.bfloat16))
    _put(s["v_pages"], s["page_table"], seq, pos, rows[:, nq + nkv:])
    return _norm_rope(rows[:, :nq], s["q_weight"], pos).to(torch.bfloat16), s["k_pages"], s["v_pages"]


def _plain_prefill(s):
    c = s["case"]
    nq, nkv, b = c["nq"], c["nkv"], s["page_table"].shape[0]
    seq, at, pos = _places(s)
    n = s["longest"]
    q = torch.zeros(b, n, nq, HD, device=pos.device)
    q[seq, at] = s["q"].float()
    q = q.view(b, n, nkv, nq // nkv, HD).permute(0, 2, 3, 1, 4)
    where = torch.zeros(b, n, dtype=torch.long, device=pos.device)  # rows that only pad see the first key
    where[seq, at] = pos
    keys, values = _held(s["k_pages"], s["page_table"]), _held(s["v_pages"], s["page_table"])
    o = _attend(q, keys, values, _sees(where, keys.shape[2], c["window"], c["sinks"]))
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, nq * HD)[seq, at].to(torch.bfloat16)


def _plain_copy(s):
    dev = s["pages"].device
    s["pages"][:, s["dst"].to(dev).long()] = s["pages"][:, s["src"].to(dev).long()]
    return s["pages"]


def _plain_logprobs(s):
    x = s["logits"].float()
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1)
    log_total = total.log()
    entropy = log_total - (e * d).sum(-1) / total
    given = d.gather(-1, s["tokens"][:, None])[:, 0] - log_total
    # keys that order the values, equal ones by the lower index first
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * (1 << 32) + ((1 << 31) - torch.arange(x.shape[1], device=x.device))
    top = key.topk(s["case"]["top"], -1).values
    ids = (1 << 31) - (top & 0xffffffff)
    return given, entropy, d.gather(-1, ids) - log_total[:, None], ids


_OWN = {"decode": _own_decode, "prefill": _own_prefill, "store": _own_store, "copy": _own_copy, "logprobs": _own_logprobs}
_PLAIN = {"decode": _plain_decode, "prefill": _plain_prefill, "store": _plain_store, "copy": _plain_copy,
          "logprobs": _plain_logprobs}


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


def _one_sequence(q, pos, k, v, case):
    """q [rows, heads, 128] of one sequence at pos against its keys and values [kv heads, keys, 128]."""
    group = q.shape[1] // k.shape[0]
    at = torch.arange(k.shape[1], device=q.device)
    out = torch.empty_like(q)
    for r in range(0, q.shape[0], 1024):
        p = pos[r:r + 1024, None]
        hidden = at > p
        if case["window"]:
            hidden |= (at <= p - case["window"]) & (at >= case["sinks"])
        for h in range(q.shape[1]):
            w = q[r:r + 1024, h] @ k[h // group].T / math.sqrt(HD)
            w[hidden] = -math.inf
            out[r:r + 1024, h] = torch.softmax(w, -1) @ v[h // group]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "copy":
        pages = s["pages"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pages[:, b] = s["pages"][:, a]
        return pages
    if op == "logprobs":
        parts = []
        for r in range(0, case["rows"], 256):
            x = s["logits"][r:r + 256].double()
            lp = torch.log_softmax(x, -1)
            ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            parts.append((lp.gather(-1, s["tokens"][r:r + 256, None])[:, 0], -(lp.exp() * lp).sum(-1), lp.gather(-1, ids), ids))
        return tuple(torch.cat(p) for p in zip(*parts))
    nq, nkv, ps = case["nq"], case["nkv"], case["page"]
    cu = list(range(case["seqs"] + 1)) if op == "decode" else s["cu_seqlens"].tolist()
    total = (s["positions"] + 1).tolist() if op == "decode" else s["kv_lens"].tolist()
    table = s["page_table"].tolist()
    outs = []
    for b in range(case["seqs"]):
        n = cu[b + 1] - cu[b]
        p = torch.arange(total[b] - n, total[b], device="cuda")
        pages = torch.tensor([x for x in table[b] if x >= 0], device="cuda")
        if op == "prefill":
            q = s["q"][cu[b]:cu[b + 1]].double()
        else:
            rows = s["qkv"][cu[b]:cu[b + 1]].view(n, nq + 2 * nkv, HD)
            q = _turn(rows[:, :nq], s["q_weight"], p)
            # the cache holds the new keys in its own type
            k = _turn(rows[:, nq:nq + nkv], s["k_weight"], p).to(torch.bfloat16)
            for j in range(nkv):
                s["k_pages"][pages[p // ps], j, p % ps] = k[:, j]
                s["v_pages"][pages[p // ps], j, p % ps] = rows[:, nq + nkv + j]
        if op == "store":
            outs.append(q)
            continue
        k, v = (s[x][pages].transpose(0, 1).reshape(nkv, -1, HD)[:, :total[b]].double() for x in ("k_pages", "v_pages"))
        outs.append(_one_sequence(q, p, k, v, case).reshape(n, nq * HD))
    out = torch.cat(outs)
    return out if op == "prefill" else (out, s["k_pages"], s["v_pages"])
