"""Drafts from the text itself (host only), and what the C entries and Python
calls of drafted decoding refuse before they touch a GPU."""

import ctypes
import random

import pytest
import torch

from nki_moe_b200 import _lib, ops
from nki_moe_b200.drafts import LookupDrafts
from nki_moe_b200.paged import PageTables


def paths(tokens, parents):
    out = []
    for i, p in enumerate(parents):
        assert -1 <= p < i
        out.append((out[p] if p >= 0 else []) + [tokens[i]])
    return out


def test_the_last_repetition_comes_first_and_others_branch_off():
    d = LookupDrafts([1, 2, 3, 4, 5, 1, 2, 3, 9, 8, 1, 2, 3])
    tokens, parents = d.tree(6)
    assert (tokens, parents) == ([9, 8, 1, 2, 3, 4], [-1, 0, 1, 2, 3, -1])
    assert d.tree(0) == ([], []) and LookupDrafts().tree(5) == ([], []) and LookupDrafts([1, 2]).tree(5) == ([], [])
    assert LookupDrafts([7, 7, 7]).tree(4) == ([7, 7], [-1, 0])
    d.extend([4])
    assert d.tree(3)[0][0] == 5
    with pytest.raises(ValueError):
        LookupDrafts([1], longest=0)


@pytest.mark.parametrize("seed", range(5))
def test_every_path_has_followed_the_text_before(seed):
    rng = random.Random(seed)
    text = [rng.randrange(4) for _ in range(rng.randrange(1, 200))]
    d = LookupDrafts(text[:50])
    d.extend(text[50:])
    for nodes in (1, 2, 7, 40, 63):
        tokens, parents = d.tree(nodes)
        assert len(tokens) == len(parents) <= nodes
        children = set(zip(parents, tokens))
        assert len(children) == len(tokens)  # no node has two children of one token
        for path in paths(tokens, parents):
            whole = [text[-1]] + path
            assert any(text[i:i + len(whole)] == whole for i in range(len(text) - len(path)))
        if text[-1] in text[:-1]:
            assert tokens


def test_sequences_know_which_pages_are_their_own():
    t = PageTables(10, 16, 6)
    a = t.add()
    t.extend([a], [40])
    assert t.alone(a, 0)
    b = t.fork(a)
    assert not t.alone(a, 0) and not t.alone(a, 39) and t.alone(a, 48)
    t.extend([a], [4])  # the last page becomes its own
    assert t.alone(a, 40) and t.alone(b, 40) and not t.alone(b, 16)


def refused(name, *args):
    with pytest.raises(_lib.NKIMoEError) as e:
        _lib.call(name, *args)
    return e.value.code


def test_the_c_entries_refuse():
    n = ctypes.c_void_p(0)
    x = ctypes.c_void_p(0x1000)  # never read: every call here ends before a launch
    inv, uns, ws = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE

    def tree(qkv=x, parents=x, nh=32, nkv=4, hd=128, T=8, B=2, page=16, pages=10, mp=4, stride=None, out=x, wsz=0,
             theta=1e6, scale=0.1, window=0, wdt=_lib.BF16, k=x):
        st = page * nkv * 128 if stride is None else stride
        return refused("nkimoe_paged_tree_attention", qkv, x, x, wdt, parents, x, x, k, x, st, st, pages, page, x, mp, mp,
                       out, T, B, nh, nkv, hd, theta, 1e-6, scale, window, 0, x, wsz, n)

    assert tree() == ws
    assert tree(qkv=n) == tree(parents=n) == tree(out=n) == tree(k=n) == inv
    assert tree(nh=30) == tree(nh=0) == tree(T=-1) == tree(scale=0.0) == tree(window=-1) == tree(theta=0.0) == inv
    assert tree(wdt=_lib.I32) == tree(stride=8) == tree(qkv=ctypes.c_void_p(0x1008)) == inv
    assert tree(hd=64) == tree(nh=68) == tree(page=24) == tree(T=1 << 25) == tree(B=1 << 21) == uns
    assert tree(mp=1 << 24, B=1 << 10) == uns
    _lib.call("nkimoe_paged_tree_attention", n, n, n, _lib.BF16, n, n, n, n, n, 0, 0, 0, 16, n, 0, 0, n, 0, 0, 32, 4, 128,
              1e6, 1e-6, 0.1, 0, 0, n, 0, n)  # no rows: nothing to do
    size = _lib.size_call("nkimoe_paged_tree_attention_workspace_bytes", 64, 8, 32, 4, 41, 16)
    assert size > 64 * 2 * 32 * 128 * 2 and _lib.size_call("nkimoe_paged_tree_attention_workspace_bytes", 64, 8, 32, 5, 4, 16) == 0

    def sample(logits=x, dt=_lib.F32, u=x, udt=_lib.F32, t=1.0, k=0, p=1.0, m=0.0, rows=2, vocab=10, tok=x, lp=x):
        return refused("nkimoe_sample_tokens", logits, dt, vocab, u, udt, n, t, n, k, n, p, n, m, rows, vocab, tok, lp, n)

    assert sample(logits=n) == sample(u=n) == sample(tok=n) == sample(lp=n) == sample(vocab=0) == sample(rows=-1) == inv
    assert sample(t=-1.0) == sample(t=float("nan")) == sample(t=float("inf")) == sample(k=-1) == inv
    assert sample(p=1.1) == sample(p=float("nan")) == sample(m=-0.1) == sample(m=1.5) == inv
    assert sample(tok=ctypes.c_void_p(0x1004)) == sample(logits=ctypes.c_void_p(0x1002)) == inv
    assert sample(dt=_lib.I32) == sample(udt=_lib.BF16) == sample(vocab=(1 << 18) + 1) == sample(rows=1 << 26) == uns
    _lib.call("nkimoe_sample_tokens", n, _lib.F32, 10, n, _lib.F64, n, 1.0, n, 0, n, 1.0, n, 0.0, 0, 10, n, n, n)

    def accept(tok=x, par=x, pages=x, planes=2, num=10, heads=4, page=16, row=256, ts=4, mp=4, T=8, B=2, counts=x, new=x):
        return refused("nkimoe_accept_drafts", tok, x, par, x, x, pages, planes, num, heads, page, row, x, ts, mp, counts, x,
                       new, T, B, x, n)

    assert accept(tok=n) == accept(par=n) == accept(pages=n) == accept(counts=n) == accept(new=n) == inv
    assert accept(planes=0) == accept(num=0) == accept(mp=0) == accept(ts=3) == accept(T=-1) == inv
    assert accept(pages=ctypes.c_void_p(0x1008)) == accept(new=ctypes.c_void_p(0x1004)) == inv
    assert accept(row=24) == accept(B=65536) == accept(planes=1 << 21) == accept(mp=1 << 27) == uns


def test_the_python_calls_refuse_host_tensors():
    z, i = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.sample_tokens(z, torch.zeros(4))
    with pytest.raises(ValueError):
        ops.accept_drafts(i.long(), i.long(), i, i, i[:3], z.view(1, 1, 4, 10), i.view(1, 4))
    with pytest.raises(ValueError):
        ops.paged_tree_attention(z.bfloat16(), z, z, i, i, i[:3], z, z, i.view(1, 4), 1, 1)


def test_marks_end_with_the_positions_they_are_of():
    t = PageTables(10, 16, 6)
    a = t.add()
    t.extend([a], [20])
    m = t.mark(a)
    assert t.kept(a, m) and not t.kept(a, m + 1) and not t.kept(7, m)
    t.extend([a], [5])
    assert not t.kept(a, m)
    b = t.fork(a)
    t.take_back([a], [20])  # what came behind is gone, the marked ones never were
    assert t.kept(a, m) and not t.kept(b, m)
    t.compact()
    t.trim(a)
    with pytest.raises(RuntimeError):
        t.extend([a, b], [70, 70])  # nothing was changed
    assert t.kept(a, m)
    n = t.mark(a)
    t.take_back([a], [19])
    t.extend([a], [1])  # as long as before
    assert not t.kept(a, m) and not t.kept(a, n)
    k = t.mark(a)
    assert t.kept(a, k)
    t.unmark(a, k)
    assert not t.kept(a, k)
    k = t.mark(a)
    t.free(a)
    assert not t.kept(a, k)
    with pytest.raises(ValueError):
        t.mark(a)
