"""Attention of trees of drafted tokens over the paged cache against the formulas
in 64 bits.

Bars.  An output is one rounding to bf16 (2^-9 of the value) of what fp32
arithmetic gives; 2^-8 leaves as much again for it.  Queries enter the tensor cores as
a sum of two bf16 (2^-17), which leaves the scores as the decode step's are
(``test_gpu_paged.py``: 2^-10 of the largest value).  Softmax weights enter rounded to
bf16: each is off by at most 2^-9 of itself, so their sum with the values is off by at
most 2^-9 of the largest value.  Together 2^-9 + 2^-10.
"""

import math
import random

import pytest
import torch

from nki_moe_b200 import ops
from nki_moe_b200._lib import NKIMoEError
from tests.test_gpu_paged import EPS, HD, Cache, near, step_inputs, turned, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def lines_of(parents):
    """Each node's path from its root."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def random_tree(n, rng):
    return [-1] + [rng.choice([i - 1, i - 1, rng.randrange(i), -1 if i % 7 == 3 else i // 2]) for i in range(1, n)][:n - 1]


def tree_case(pasts, trees, nq, nkv, ps, window=0, sinks=0, seed=0, w_dtype=torch.bfloat16, tail=0, scale=None,
              interleaved=False, missing=True):
    B = len(pasts)
    nodes = [len(t) for t in trees]
    total = [p + n for p, n in zip(pasts, nodes)]

    def needed(b, lo, hi):
        # what the root sees, and the tree
        return hi > pasts[b] or any((s > pasts[b] - window) or s < sinks for s in range(lo, hi))

    c = Cache(total, nkv, ps, seed, needed if window and missing else None)
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(nodes) + tail
    qkv = torch.randn(T, (nq + 2 * nkv) * HD, generator=g).bfloat16()
    qkv[sum(nodes):] = math.nan
    qw, kw = weights(seed + 2, w_dtype)
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
    lines = [lines_of(t) for t in trees]
    pos = torch.tensor([pasts[b] + len(x) - 1 for b in range(B) for x in lines[b]], dtype=torch.int64)
    rows = qkv[:sum(nodes)].view(-1, nq + 2 * nkv, HD)
    q = turned(rows[:, :nq], qw, pos)
    new = turned(rows[:, nq:nq + nkv], kw, pos)
    grp = nq // nkv
    k_ref, v_ref = c.k.clone(), c.v.clone()
    ref = torch.zeros(sum(nodes), nq, HD, dtype=torch.float64)
    places, vmax = [], 1.0
    for b in range(B):
        for i in range(nodes[b]):
            s, r = pasts[b] + i, int(cu[b]) + i
            pg = int(c.table[b, s // ps])
            k_ref[pg, :, s % ps], v_ref[pg, :, s % ps] = new[r].bfloat16(), rows[r, nq + nkv:]
            places.append((pg, s % ps))
    for b in range(B):
        k, v = c.rows(k_ref, b, total[b]), c.rows(v_ref, b, total[b])
        vmax = max(vmax, float(v.nan_to_num().abs().max())) if total[b] else vmax
        for i in range(nodes[b]):
            r = int(cu[b]) + i
            p = int(pos[r])
            at = torch.arange(total[b])
            see = at < pasts[b]
            if window:
                see &= (at > p - window) | (at < sinks)
            for d, a in enumerate(lines[b][i]):
                see[pasts[b] + a] = not window or pasts[b] + d > p - window or pasts[b] + d < sinks
            for h in range(nq):
                w = torch.softmax((k[h // grp][see] @ q[r, h]) * (scale or HD ** -0.5), 0)
                ref[r, h] = w @ v[h // grp][see]
    if interleaved:
        pool = torch.stack([c.k, c.v], 1).cuda()
        kd, vd = pool[:, 0], pool[:, 1]
    else:
        kd, vd = c.k.cuda(), c.v.cuda()
    before_k, before_v = kd.clone(), vd.clone()
    flat = torch.tensor([p for t in trees for p in t] + [99] * tail, dtype=torch.int32)
    kv = torch.tensor(total, dtype=torch.int32)
    out = torch.full((T, nq * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    args = [qkv.cuda(), qw.cuda(), kw.cuda(), flat.cuda(), cu.cuda(), kv.cuda(), kd, vd, c.table.cuda(), nq, nkv]
    got = ops.paged_tree_attention(*args, window=window, sinks=sinks, scale=scale, out=out)
    ops.read_paged_status()
    assert got is out and (out[sum(nodes):] == 7.0).all()  # rows of no sequence stay
    res = out[:sum(nodes)].view(-1, nq, HD)
    near(res, ref, vmax, atol=2 ** -9 + 2 ** -10)
    # the nodes' rows in the cache, and nothing else
    for now, old, want, exact in ((kd, before_k, k_ref, False), (vd, before_v, v_ref, True)):
        now, old = now.cpu(), old.cpu()
        for pg, at in places:
            a, w = now[pg, :, at].double(), want[pg, :, at].double()
            assert torch.equal(a, w) if exact else ((a - w).abs() <= 2 ** -7 * w.abs() + 2 ** -13).all()
            now[pg, :, at] = old[pg, :, at]
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))
    return args, out


def trees_of(sizes, seed=0):
    rng = random.Random(seed)
    return [random_tree(n, rng) if n else [] for n in sizes]


@pytest.mark.parametrize("nq,nkv", [(32, 4), (8, 8), (16, 1), (12, 4), (7, 1), (40, 8), (18, 2)])
@pytest.mark.parametrize("ps", [16, 64])
def test_heads_and_small_trees(nq, nkv, ps):
    tree_case([0, 1, 15, 63, 64, 128, 300], trees_of([1, 2, 5, 8, 3, 7, 4], nq), nq, nkv, ps, seed=nq + ps)


@pytest.mark.parametrize("nq,nkv", [(32, 4), (16, 1), (8, 8), (12, 4)])
def test_trees_of_all_sizes(nq, nkv):
    tree_case([100, 0, 37, 250, 90, 127], trees_of([16, 17, 33, 9, 64, 32], nq), nq, nkv, 32, seed=nq)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_page_sizes(ps):
    tree_case([ps - 1, ps, 3 * ps + 7, 500], trees_of([4, 40, 13, 2], ps), 16, 2, ps, seed=ps)


@pytest.mark.parametrize("past", [0, 1, 120, 128, 191, 1000])
@pytest.mark.parametrize("shape", ["chain", "star", "roots"])
def test_shapes(past, shape):
    n = 40
    tree = {"chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1), "roots": [-1] * n}[shape]
    tree_case([past, past + 3], [tree, tree[:11]], 16, 2, 16, seed=past + len(shape))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 0), (3, 2), (16, 4), (64, 4), (100, 65), (17, 300), (1000, 4),
                                          (700, 0)])
def test_window_and_sinks(window, sinks):
    tree_case([0, 2, 64, 100, 333, 700], trees_of([9, 12, 1, 30, 5, 14], window), 32, 4, 16, window, sinks, seed=window + sinks)


def test_window_within_chains():
    """Ancestors that the window has passed are not seen, first positions are."""
    chain = list(range(-1, 39))
    for window, sinks in ((5, 0), (5, 3), (20, 8), (39, 1)):
        tree_case([0, 4, 130], [chain, chain[:12], chain], 16, 2, 16, window, sinks, seed=window)


def test_long_sequences_are_split_over_the_gpu():
    tree_case([20011], trees_of([13], 1), 32, 4, 64, seed=5)
    tree_case([9000], trees_of([50], 2), 16, 1, 128, seed=6)


def test_ragged_batch():
    tree_case([1, 5000, 40, 2, 1200, 64, 0, 3000], trees_of([8, 3, 20, 1, 64, 16, 5, 11], 3), 16, 2, 32, seed=7)


def test_sequences_without_nodes_and_rows_of_no_sequence():
    tree_case([30, 5, 64, 0, 9], trees_of([0, 4, 0, 0, 18], 4), 16, 2, 16, seed=8, tail=21)


def test_fp32_weights_interleaved_pools_and_scale():
    tree_case([5, 70, 129], trees_of([6, 24, 2], 5), 16, 2, 16, seed=9, w_dtype=torch.float32, interleaved=True, scale=0.05)


def test_many_sequences_in_one_workspace():
    """Counters and parts of one call must not disturb the next."""
    for i, (pasts, sizes, nq, nkv) in enumerate([([3000], [12], 16, 2), ([70] * 300, [2] * 300, 8, 2), ([5000, 1], [3, 64], 16, 1),
                                                 ([65] * 40, [5] * 40, 8, 8), ([3000], [12], 16, 2)]):
        tree_case(pasts, trees_of(sizes, i), nq, nkv, 64, seed=20 + i)


def test_more_rows_than_ctas():
    """From 4 * 148 rows on a warp stores a row by itself."""
    tree_case([40] * 30, trees_of([21] * 30, 6), 8, 2, 16, seed=40)


def test_one_node_is_a_decode_step():
    """Bit for bit in the cache, to rounding in the output."""
    a = step_inputs([70, 33, 500, 1], 16, 2, 16, 50)
    b = [t.clone() if isinstance(t, torch.Tensor) else t for t in a]
    want = ops.paged_decode_attention(*a)
    n = 4
    out = ops.paged_tree_attention(b[0], b[1], b[2], torch.full((n,), -1, dtype=torch.int32, device="cuda"),
                                   torch.arange(n + 1, dtype=torch.int32, device="cuda"), (b[3] + 1).int(), *b[4:])
    ops.read_paged_status()
    for x, y in zip(a[4:6], b[4:6]):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    assert ((out.double() - want.double()).abs() <= 2 ** -7 * want.double().abs() + 2 ** -9).all()


def test_deterministic_streams_and_graphs():
    args, out = tree_case([2000, 37, 800, 1], trees_of([9, 3, 30, 16], 7), 32, 4, 16, seed=51)
    want = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.paged_tree_attention(*args) for _ in range(3)]
    here = [ops.paged_tree_attention(*args) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + here)
    graphs = []
    for seed in (52, 53):  # captured on one stream, replayed on two
        a, o = tree_case([4000, 900, 65], trees_of([9, 3, 33], seed), 16, 2, 64, seed=seed)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = ops.paged_tree_attention(*a)
        graphs.append((g, a, got, o.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        ops.paged_tree_attention(*args)
    torch.cuda.synchronize()
    for _, _, got, o in graphs:
        assert torch.equal(got, o)
    # lengths and trees are device data: a replay serves the next step
    g, a, got, _ = graphs[0]
    a[3].copy_(torch.tensor([-1] * a[3].numel(), dtype=torch.int32))
    a[5].sub_(40)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, ops.paged_tree_attention(*a))
    ops.read_paged_status()


def test_bad_data_is_reported(monkeypatch):
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    args, out = tree_case([70, 33, 50], trees_of([6, 5, 7], 8), 8, 2, 16, seed=54)
    good = out.clone()

    def run(i, bad):
        call = list(args)
        call[i] = bad
        call[6], call[7] = args[6].clone(), args[7].clone()  # lengths that overlap write other places
        out.fill_(3.0)
        ops.paged_tree_attention(*call, out=out)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
        ops.read_paged_status()  # cleared
        return out

    # a parent that does not come before its child: a root
    for value in (5, 1, -2, 10 ** 9):
        parents = args[3].clone()
        parents[6 + 1] = value
        got = run(3, parents)
        parents[6 + 1] = -1
        call = list(args)
        call[3] = parents
        assert torch.equal(got, ops.paged_tree_attention(*call))
    # lengths: their rows stay
    for b, value in ((0, 2), (1, 10 ** 6), (2, -1)):
        kv = args[5].clone()
        kv[b] = value
        got = run(5, kv)
        cu = args[4].tolist()
        for q in range(3):
            part = got[cu[q]:cu[q + 1]]
            assert (part == 3.0).all() if q == b else torch.equal(part, good[cu[q]:cu[q + 1]])
    got = run(4, torch.tensor([0, 6, 6 - 2, 18], dtype=torch.int32, device="cuda"))
    got = run(4, torch.tensor([0, 6, 11, 400], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[:11], good[:11])
    # rows that the call does not have, within what a tree may hold
    got = run(4, torch.tensor([0, 6, 11, 18 + 40], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[:11], good[:11]) and (got[11:] == 3.0).all()
    got = run(4, torch.tensor([-30, 6, 11, 18], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[6:], good[6:]) and (got[:6] == 3.0).all()
    # a page that the tree needs
    for bad in (-1, 10 ** 6):
        table = args[8].clone()
        table[1, 0] = bad
        got = run(8, table)
        assert torch.equal(got[:6], good[:6]) and torch.equal(got[11:], good[11:])


def test_more_than_64_nodes_are_reported():
    nq, nkv = 8, 2
    c = Cache([200, 90], nkv, 16, 55)
    T = 65 + 4
    g = torch.Generator().manual_seed(55)
    qkv = torch.randn(T, (nq + 2 * nkv) * HD, generator=g).bfloat16().cuda()
    qw, kw = (w.cuda() for w in weights(55))
    cu = torch.tensor([0, 65, 69], dtype=torch.int32, device="cuda")
    kv = torch.tensor([200, 90], dtype=torch.int32, device="cuda")
    out = torch.full((T, nq * HD), 3.0, dtype=torch.bfloat16, device="cuda")
    parents = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    ops.paged_tree_attention(qkv, qw, kw, parents, cu, kv, c.k.cuda(), c.v.cuda(), c.table.cuda(), nq, nkv, out=out)
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    assert (out[:65] == 3.0).all() and torch.isfinite(out[65:]).all() and not (out[65:] == 3.0).all()


def test_pool_past_32_bit_offsets():
    nq, nkv, ps = 8, 4, 256
    P = 2 ** 31 // (nkv * ps * HD) + 40
    k = torch.zeros(P, nkv, ps, HD, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    args, out = tree_case([590, 300], trees_of([10, 4], 9), nq, nkv, ps, seed=56)
    first = P - args[6].shape[0]
    k[first:], v[first:] = args[6], args[7]
    table = torch.where(args[8] >= 0, args[8] + first, args[8])
    big = ops.paged_tree_attention(*args[:6], k, v, table, nq, nkv)
    ops.read_paged_status()
    assert torch.equal(big, out)


def test_refusals():
    args, out = tree_case([20, 30], trees_of([4, 3], 10), 8, 2, 16, seed=57)
    for i, bad in ((0, args[0].float()), (0, args[0][:, :-128]), (0, args[0].cpu()), (0, args[0].t()), (1, args[1][:64]),
                   (3, args[3].long()), (3, args[3][:5]), (3, args[3].cpu()), (4, args[4].long()), (4, args[4][:2]),
                   (5, args[5].cpu()), (6, args[6].float()), (6, args[6][:, :, :8]), (7, args[7][:-1]),
                   (8, args[8][:1]), (8, args[8].long()), (9, 9), (10, 3)):
        call = list(args)
        call[i] = bad
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_tree_attention(*call)
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=math.inf), dict(theta=-1.0),
               dict(out=out.float()), dict(out=out[:3]), dict(out=args[0].view(-1)[:out.numel()].view(out.shape))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_tree_attention(*args, **kw)
    empty = torch.empty(0, args[0].shape[1], dtype=torch.bfloat16, device="cuda")
    none = ops.paged_tree_attention(empty, args[1], args[2], args[3][:0], torch.zeros(3, dtype=torch.int32, device="cuda"),
                                    args[5], *args[6:])
    assert none.shape == (0, 8 * HD)
    assert EPS == 1e-6
