"""Acceptance of drafted tokens on the GPU against the walk written out.
Everything is whole numbers or copies: results have to be equal."""

import random

import pytest
import torch

from nki_moe_b200 import ops
from nki_moe_b200._lib import NKIMoEError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def walk(tokens, sampled, parents):
    path = [0] if tokens else []
    while path:
        nxt = [i for i in range(path[-1] + 1, len(tokens)) if parents[i] == path[-1] and tokens[i] == sampled[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


def tree(n, rng, vocab):
    parents = [-1] + [rng.choice([i - 1, rng.randrange(i)]) for i in range(1, n)]
    return [rng.randrange(vocab) for _ in range(n)], [rng.randrange(vocab) for _ in range(n)], parents[:n]


def case(nodes, pasts, seed, vocab=3, lead=(2, 3), nkv=2, ps=16, hd=128, dtype=torch.bfloat16, tail=0, trees=None):
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    trees = trees or [tree(n, rng, vocab) for n in nodes]
    need = [-(-(p + n) // ps) for p, n in zip(pasts, nodes)]
    P = sum(need) + 2
    ids = torch.randperm(P, generator=g)[:sum(need)].tolist()
    table = torch.full((len(nodes), max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    pages = torch.randint(-128, 127, (*lead, P, nkv, ps, hd), generator=g, dtype=torch.int8)
    pages = pages.to(dtype) if dtype != torch.int8 else pages
    cu = torch.tensor([0] + nodes).cumsum(0).to(torch.int32)
    T = int(cu[-1]) + tail
    flat = [sum((t[i] for t in trees), []) + [0] * tail for i in range(3)]
    kv = torch.tensor([p + n for p, n in zip(pasts, nodes)], dtype=torch.int32)
    want, counts = pages.clone(), []
    path, new = torch.full((T,), -1, dtype=torch.int32), torch.full((T,), -1)
    for b, (tok, sam, par) in enumerate(trees):
        w = walk(tok, sam, par)
        counts.append(len(w))
        for k, i in enumerate(w):
            f, d = pasts[b] + i, pasts[b] + k
            want[..., int(table[b, d // ps]), :, d % ps, :] = pages[..., int(table[b, f // ps]), :, f % ps, :]
            path[cu[b] + k], new[cu[b] + k] = i, sam[i]
    args = [torch.tensor(flat[0]), torch.tensor(flat[1]), torch.tensor(flat[2], dtype=torch.int32), cu, kv, pages, table]
    return args, (torch.tensor(counts, dtype=torch.int32), path, new, want)


def check(args, want):
    dev = [a.cuda() for a in args]
    counts, path, new = ops.accept_drafts(*dev)
    ops.read_paged_status()
    for got, ref in zip((counts, path, new, dev[5]), want):
        assert got.dtype == ref.dtype and torch.equal(got.cpu(), ref)
    return dev


@pytest.mark.parametrize("vocab", [1, 2, 3, 50])
@pytest.mark.parametrize("ps", [16, 64])
def test_trees_of_all_sizes(vocab, ps):
    nodes = [1, 2, 3, 7, 8, 31, 32, 33, 34, 63, 64]
    check(*case(nodes, [0, 1, 15, 16, 17, 40, 63, 64, 5, 0, 100], vocab + ps, vocab, ps=ps))


def test_chains():
    """A chain that is agreed with as a whole, in part, not at all: nothing moves."""
    trees = []
    for agree in (64, 33, 32, 31, 1):
        par = list(range(-1, 63))
        trees.append(([7] * 64, [7] * (agree - 1) + [8] * (65 - agree), par))
    args, want = case([64] * 5, [3] * 5, 1, trees=trees)
    assert want[0].tolist() == [64, 33, 32, 31, 1] and torch.equal(want[3], args[5])
    check(args, want)


def test_moves_over_long_paths():
    """Every second node is on the path: places are read and written again within one move."""
    tok = [5] * 64
    sam = [5] * 64
    par = [-1] + [0] * 63
    for i in range(2, 64, 2):
        par[i] = i - 2
    tok[1::2] = [9] * 32
    args, want = case([64, 64], [11, 32], 2, trees=[(tok, sam, par)] * 2)
    assert want[0].tolist() == [32, 32]
    check(args, want)


@pytest.mark.parametrize("lead,nkv,hd,dtype", [((), 1, 16, torch.int8), ((1,), 4, 128, torch.bfloat16),
                                               ((48, 2), 4, 128, torch.bfloat16), ((3,), 8, 64, torch.float32),
                                               ((7,), 3, 8, torch.bfloat16)])
def test_pools_of_other_shapes(lead, nkv, hd, dtype):
    check(*case([9, 20, 1], [30, 7, 50], 3, 2, lead=lead, nkv=nkv, hd=hd, dtype=dtype))


def test_odd_trees():
    """Two roots, parents that come later or make no sense, equal drafts of one node: the lowest counts."""
    trees = [([1, 2, 2, 3, 3], [2, 3, 3, 9, 9], [-1, 0, 0, 2, 1]),  # 0 -> 1 -> 4, not 2 -> 3
             ([1, 2, 3], [2, 3, 4], [-1, -1, 1]),  # the second root is never reached
             ([1, 2, 3], [3, 2, 2], [-1, 2, 0]),  # node 1 names a later parent: 0 -> 2, and 1 is not above 2
             ([1, 2, 2], [2, 5, 2], [-1, 1, 0]),  # node 1 is its own parent
             ([1, 2, 3], [2, 3, 4], [-7, 99, -2])]
    args, want = case([5, 3, 3, 3, 3], [4, 4, 20, 0, 1], 4, trees=trees)
    assert want[0].tolist() == [3, 1, 2, 2, 1]
    check(args, want)


def test_sequences_without_nodes_and_rows_of_no_sequence():
    check(*case([0, 4, 0, 0, 6, 0], [5, 9, 0, 40, 31, 1], 5, 1, tail=37))


def test_many_sequences():
    rng = random.Random(6)
    nodes = [rng.randrange(1, 20) for _ in range(500)]
    check(*case(nodes, [rng.randrange(100) for _ in nodes], 6, 2, lead=(2,), nkv=1, hd=8))


def test_bad_lengths_and_pages_are_reported():
    args, want = case([4, 65, 4], [10, 3, 14], 7, 1, trees=[([1] * 4, [1] * 4, [-1, 0, 0, 2])] + [([1] * 65, [1] * 65, [-1] * 65)]
                      + [([1, 9, 1, 1], [1] * 4, [-1, 0, 0, 2])])
    counts, path, _, pages = want
    dev = [a.cuda() for a in args]
    got = ops.accept_drafts(*dev)
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    assert got[0].tolist() == [2, 0, 3]  # 65 nodes are too many
    assert torch.equal(dev[5].cpu()[..., :, :, :], pages)
    # a page that a moved row needs is not held
    args, want = case([4], [14], 8, 1, trees=[([1, 9, 1, 1], [1] * 4, [-1, 0, 0, 2])])
    for bad in (-1, 10 ** 6):
        dev = [a.cuda() for a in args]
        dev[6][0, 1] = bad
        got = ops.accept_drafts(*dev)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
        assert got[0].tolist() == [3] and got[1].tolist() == [0, 2, 3, -1]
        assert torch.equal(dev[5].cpu(), args[5])  # both rows come from that page
    for cu, kv in (([0, 9], [18]), ([-1, 4], [18]), ([3, 1], [18]), ([0, 4], [3]), ([0, 4], [1000])):
        dev = [a.cuda() for a in args]
        dev[3], dev[4] = torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor(kv, dtype=torch.int32).cuda()
        got = ops.accept_drafts(*dev)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
        assert got[0].tolist() == [0] and torch.equal(dev[5].cpu(), args[5])


def test_graph_replays_with_new_trees():
    args, want = case([8] * 4, [20, 3, 40, 15], 9, 2)
    dev = check(args, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.accept_drafts(*dev)
    for seed in (10, 11):
        args, want = case([8] * 4, [20, 3, 40, 15], seed, 2)
        for d, a in zip(dev, args):
            d.copy_(a)
        g.replay()
        torch.cuda.synchronize()
        for x, ref in zip((*got, dev[5]), want):
            assert torch.equal(x.cpu(), ref)


def test_refusals():
    args, _ = case([4, 4], [3, 9], 12)
    dev = [a.cuda() for a in args]
    ops.accept_drafts(*dev)
    for i, bad in ((0, dev[0].int()), (0, dev[0][:5]), (1, dev[1].cpu()), (1, dev[1].float()), (2, dev[2].long()),
                   (3, dev[3].long()), (3, dev[3][:2]), (4, dev[4].cpu()), (5, dev[5][..., :-1]), (5, dev[5].cpu()),
                   (5, dev[5][0, 0, 0]), (6, dev[6].long()), (6, dev[6][:1]), (6, dev[6].cpu()),
                   (5, torch.zeros(4, 1, 16, 5, device="cuda"))):
        call = list(dev)
        call[i] = bad
        with pytest.raises((ValueError, RuntimeError)):
            ops.accept_drafts(*call)
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    out = ops.accept_drafts(empty, empty, empty.int(), torch.zeros(3, dtype=torch.int32, device="cuda"),
                            torch.zeros(2, dtype=torch.int32, device="cuda"), dev[5], dev[6])
    assert out[0].tolist() == [0, 0] and out[1].numel() == out[2].numel() == 0
