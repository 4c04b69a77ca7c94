"""The bookkeeping of the paged cache (host only), and what the C ABI and the
Python entry points refuse before they touch a GPU."""

import ctypes
import random

import pytest
import torch

from nki_moe_b200 import _lib, ops
from nki_moe_b200.paged import CacheFull, PagedKVCache, PageTables


def test_extend_takes_the_lowest_pages_and_counts_lengths():
    t = PageTables(8, 16, 4)
    a, b = t.add(), t.add()
    assert t.extend([a, b], [17, 16]) == []
    assert t.pages(a) == [0, 1] and t.pages(b) == [2] and t.length(a) == 17 and t.free_pages == 5
    assert t.extend([b, a], [1, 15]) == []
    assert t.pages(b) == [2, 3] and t.pages(a) == [0, 1] and t.length(a) == 32
    t.free(a)
    assert t.free_pages == 6 and a not in t
    c = t.add()
    t.extend([c], [1])
    assert t.pages(c) == [0]
    assert t.table([c, b]).tolist() == [[0, -1, -1, -1], [2, 3, -1, -1]]


def test_extend_refuses_without_changing_anything():
    t = PageTables(3, 16, 2)
    a, b = t.add(), t.add()
    t.extend([a], [20])
    for seqs, counts, error in (([a, b], [1, 33], ValueError), ([a, a], [1, 1], ValueError), ([a], [-1], ValueError),
                                ([a], [1, 2], ValueError), ([99], [1], ValueError), ([b, a], [17, 0], CacheFull)):
        with pytest.raises(error):
            t.extend(seqs, counts)
        assert t.length(a) == 20 and t.length(b) == 0 and t.free_pages == 1
    for args in ((0, 16, 1), (4, 24, 1), (4, 16, 0), (4, 16, 1, -1), (4, 16, 1, 1, -1)):
        with pytest.raises(ValueError):
            PageTables(*args)
    with pytest.raises(ValueError):
        t.free(99)


def test_forks_share_pages_and_copy_the_last_one_when_written():
    t = PageTables(10, 16, 4)
    a = t.add()
    t.extend([a], [24])
    b, c = t.fork(a), t.fork(a)
    assert t.pages(b) == t.pages(c) == [0, 1] and t.free_pages == 8
    # two of the three write: two copies; the third keeps the page
    copies = t.extend([a, b], [1, 1])
    assert copies == [(1, 2), (1, 3)]
    assert t.pages(a) == [0, 2] and t.pages(b) == [0, 3] and t.pages(c) == [0, 1]
    assert t.extend([c], [1]) == []
    # all the sharers at once: the last keeps it
    d = t.fork(c)
    assert t.extend([c, d], [1, 1]) == [(1, 4)]
    assert t.pages(d) == [0, 1] and t.pages(c) == [0, 4]
    # a full last page is not written: nothing to copy
    t.extend([d], [6])
    e = t.fork(d)
    assert t.length(d) == 32 and t.extend([d, e], [1, 1]) == []
    for q in (a, b, c, d, e):
        t.free(q)
    assert t.free_pages == 10


def test_trim_gives_back_what_a_window_has_passed():
    t = PageTables(20, 16, 20, window=20, sinks=17)
    a = t.add()
    t.extend([a], [100])
    # position 100 sees 81 .. 100 and 0 .. 16: pages 0, 1 and from 5 on
    assert t.trim(a) == 3 and t.pages(a) == [0, 1, -1, -1, -1, 5, 6] and t.trim(a) == 0
    b = t.fork(a)
    t.extend([a, b], [1, 1])
    t.free(a)
    t.free(b)
    assert t.free_pages == 20
    t = PageTables(4, 16, 4, window=1)
    a = t.add()
    t.extend([a], [32])
    assert t.trim(a) == 2 and t.pages(a) == [-1, -1] and t.extend([a], [1]) == []


def test_compact_moves_pages_to_the_front():
    t = PageTables(10, 16, 4)
    a, b, c = t.add(), t.add(), t.add()
    t.extend([a, b, c], [32, 32, 40])
    d = t.fork(c)
    t.free(a)
    t.free(b)
    moves = t.compact()
    assert moves == [(4, 0), (5, 1), (6, 2)] and t.pages(c) == t.pages(d) == [0, 1, 2]
    assert t.compact() == [] and t.free_pages == 7
    t.extend([c], [1])
    assert t.pages(c) == [0, 1, 3]


def test_random_use_against_a_model_of_contents():
    """Every page's contents, copied as the tables say, always hold what the
    sequences have written."""
    rng = random.Random(7)
    t = PageTables(40, 16, 8, window=50, sinks=5)
    memory = [[None] * 16 for _ in range(40)]
    texts: dict[int, list] = {}

    def run(copies):
        assert not {a for a, _ in copies} & {b for _, b in copies} and len({b for _, b in copies}) == len(copies)
        for a, b in copies:
            memory[b] = list(memory[a])

    for step in range(3000):
        op = rng.random()
        if op < 0.15 and len(texts) < 12:
            texts[t.add()] = []
        elif op < 0.3 and texts and len(texts) < 12:
            q = rng.choice(list(texts))
            texts[t.fork(q)] = list(texts[q])
        elif op < 0.4 and texts:
            q = rng.choice(list(texts))
            t.free(q)
            del texts[q]
        elif op < 0.45:
            run(t.compact())
        elif texts:
            seqs = rng.sample(list(texts), rng.randint(1, min(5, len(texts))))
            counts = [min(rng.randint(0, 20), 128 - len(texts[q])) for q in seqs]
            try:
                run(t.extend(seqs, counts))
            except CacheFull:
                continue
            for q, n in zip(seqs, counts):
                for _ in range(n):
                    at = len(texts[q])
                    texts[q].append((q, step, at))
                    memory[t.pages(q)[at // 16]][at % 16] = texts[q][-1]
                t.trim(q)
        for q, text in texts.items():
            pages, n = t.pages(q), len(text)
            assert t.length(q) == n
            for s in range(n):
                if s < 5 or s > n - 50:
                    assert memory[pages[s // 16]][s % 16] == text[s]
    for q in list(texts):
        t.free(q)
    assert t.free_pages == 40


def test_take_back_undoes_an_extension():
    t = PageTables(8, 16, 4)
    a, b = t.add(), t.add()
    t.extend([a, b], [20, 16])
    c = t.fork(a)
    t.extend([a, b], [40, 1])  # a copies its last page
    assert t.pages(a) == [0, 3, 4, 5] and t.pages(b) == [2, 6] and t.free_pages == 1
    t.take_back([a, b], [20, 16])
    assert t.pages(a) == [0, 3] and t.length(a) == 20 and t.pages(b) == [2] and t.length(b) == 16
    assert t.pages(c) == [0, 1] and t.free_pages == 4
    t.take_back([b, c], [0, 20])
    assert t.pages(b) == [] and t.length(b) == 0 and t.free_pages == 5
    for seqs, lengths in (([a], [21]), ([a], [-1]), ([99], [0]), ([a], []), ([a, b], [20, 1])):
        with pytest.raises(ValueError):
            t.take_back(seqs, lengths)
    assert t.length(a) == 20 and t.free_pages == 5
    t.extend([b], [64])
    assert t.free_pages == 1


# ------------------------------------------------------------------ refusals
NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(4096)  # never dereferenced: the checks come first


def code(name, *args):
    with pytest.raises(_lib.NKIMoEError) as e:
        _lib.call(name, *args)
    return e.value.code


def store_args(**kw):
    a = dict(qkv=SOME, qw=SOME, kw=SOME, wdt=_lib.BF16, cu=SOME, kv=SOME, k=SOME, v=SOME, ks=8192, vs=8192, pages=4,
             ps=16, table=SOME, ts=4, mp=4, out=SOME, T=3, B=1, nq=8, nkv=4, hd=128, theta=1e6, eps=1e-6, status=SOME,
             stream=NULL)
    a.update(kw)
    return list(a.values())


def decode_args(**kw):
    a = dict(qkv=SOME, qw=SOME, kw=SOME, wdt=_lib.BF16, pos=SOME, pst=1, k=SOME, v=SOME, ks=8192, vs=8192, pages=4,
             ps=16, table=SOME, ts=4, mp=4, out=SOME, B=1, nq=8, nkv=4, hd=128, theta=1e6, eps=1e-6, scale=0.1,
             window=0, sinks=0, ws=SOME, wsb=1 << 30, stream=NULL)
    a.update(kw)
    return list(a.values())


def prefill_args(**kw):
    a = dict(q=SOME, qs=1024, k=SOME, v=SOME, ks=8192, vs=8192, pages=4, ps=16, table=SOME, ts=4, mp=4, cu=SOME,
             kv=SOME, out=SOME, T=3, B=1, nq=8, nkv=4, hd=128, scale=0.1, window=0, sinks=0, ws=SOME, wsb=1 << 30,
             stream=NULL)
    a.update(kw)
    return list(a.values())


CALLS = {"nkimoe_qk_norm_rope_store": store_args, "nkimoe_paged_decode_attention": decode_args,
         "nkimoe_paged_prefill_attention": prefill_args}


@pytest.mark.parametrize("name", list(CALLS))
def test_paged_calls_refuse_bad_arguments(name):
    args = CALLS[name]
    inv, uns = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED
    for kw, want in ((dict(ps=24), uns), (dict(ps=8), uns), (dict(ps=512), uns), (dict(hd=64), uns),
                     (dict(nq=9), inv), (dict(nq=68), uns), (dict(nq=0), inv), (dict(pages=0), inv), (dict(mp=0), inv),
                     (dict(ks=8191), inv), (dict(vs=8196), inv), (dict(ts=3), inv), (dict(k=NULL), inv),
                     (dict(table=NULL), inv), (dict(v=ctypes.c_void_p(4100)), inv), (dict(out=NULL), inv),
                     (dict(B=-1), inv), (dict(mp=1 << 27, ts=1 << 27), uns)):
        assert code(name, *args(**kw)) == want, kw
    if name != "nkimoe_qk_norm_rope_store":
        for kw, want in ((dict(window=-1), inv), (dict(sinks=-1), inv), (dict(scale=0.0), inv), (dict(scale=-1.0), inv),
                         (dict(scale=float("nan")), inv), (dict(wsb=100), _lib.ERR_WORKSPACE), (dict(ws=NULL), inv)):
            assert code(name, *args(**kw)) == want, kw
    if name == "nkimoe_paged_decode_attention":
        for kw, want in ((dict(B=5000), uns), (dict(pst=2), inv), (dict(wdt=_lib.I32), inv), (dict(pos=NULL), inv)):
            assert code(name, *args(**kw)) == want, kw
    if name == "nkimoe_paged_prefill_attention":
        for kw, want in ((dict(qs=1023), inv), (dict(qs=1028), inv), (dict(T=-1), inv), (dict(cu=NULL), inv)):
            assert code(name, *args(**kw)) == want, kw
    # nothing to do is no error
    _lib.call(name, *args(B=0, T=0) if name != "nkimoe_paged_decode_attention" else args(B=0))


def test_copies_are_checked_before_the_launch():
    ids = lambda *x: (ctypes.c_int32 * len(x))(*x)  # noqa: E731
    inv = _lib.ERR_INVALID_ARG
    for src, dst in (((0, 1), (2, 2)), ((0, 1), (1, 3)), ((5,), (0,)), ((0,), (5,)), ((-1,), (0,)), ((2,), (2,))):
        assert code("nkimoe_copy_pages", SOME, 2, 5, 4096, ids(*src), ids(*dst), len(src), NULL) == inv
    assert code("nkimoe_copy_pages", SOME, 2, 5, 4090, ids(0), ids(1), 1, NULL) == _lib.ERR_UNSUPPORTED
    assert code("nkimoe_copy_pages", NULL, 2, 5, 4096, ids(0), ids(1), 1, NULL) == inv
    assert code("nkimoe_copy_pages", SOME, 0, 5, 4096, ids(0), ids(1), 1, NULL) == inv
    _lib.call("nkimoe_copy_pages", SOME, 2, 5, 4096, NULL, NULL, 0, NULL)


def test_token_scores_refuse_bad_arguments():
    inv, uns = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED

    def go(x=SOME, dt=_lib.F32, st=100, tok=SOME, rows=2, v=100, n=5, wsb=1 << 20):
        return code("nkimoe_token_logprobs", x, dt, st, tok, rows, v, n, SOME, SOME, SOME, SOME, SOME, wsb, NULL)

    assert go(x=NULL) == inv and go(dt=_lib.I32) == uns and go(n=33) == uns and go(n=-1) == inv and go(v=3) == uns
    assert go(rows=-1) == inv and go(tok=NULL) == inv and go(x=ctypes.c_void_p(4097)) == inv
    assert go(wsb=10) == _lib.ERR_WORKSPACE


def test_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 10 * 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    pages = torch.zeros(4, 1, 16, 128, dtype=torch.bfloat16)
    table = torch.zeros(2, 2, dtype=torch.int32)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_decode_attention(x, w, w, torch.zeros(2, dtype=torch.int64), pages, pages, table, 8, 1)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_store(x, w, w, i32, i32[:2], pages, pages, table, 8, 1)
    with pytest.raises(ValueError):
        ops.paged_prefill_attention(x.view(2, 10, 128), pages, pages, table, i32, i32[:2])
    with pytest.raises(ValueError):
        ops.copy_pages(pages, [0], [1])
    with pytest.raises(ValueError):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("size", [0, -16, 24, 512])
def test_a_cache_refuses_other_page_sizes(size):
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 4, size, 64, device="cpu")


@pytest.mark.parametrize("pool", [5, 70000, 2 ** 30])
def test_pages_written_twice_or_read_and_written_are_refused_in_pools_of_any_size(pool):
    def ids(*x):
        return (ctypes.c_int32 * len(x))(*x)

    last = pool - 1
    for src, dst in (((0, 1), (2, 2)), ((0, last), (last, 3)), ((last,), (last,)), ((pool,), (0,)), ((0,), (-1,))):
        assert code("nkimoe_copy_pages", SOME, 2, pool, 4096, ids(*src), ids(*dst), len(src), NULL) == _lib.ERR_INVALID_ARG


def test_calls_run_on_the_device_of_their_tensors_in_any_order_of_arguments(monkeypatch):
    class OnSecond(torch.Tensor):
        is_cuda = True
        device = torch.device("cuda", 1)

        def get_device(self):
            return 1

    entered = []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *exc):
            return False

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    t = torch.zeros(2).as_subclass(OnSecond)
    fn = ops._on_its_device(lambda *args, **kw: len(args) + len(kw))
    for args, kw in (((t, 3), {}), ((), {"qkv": t, "n_heads": 8}), ((), {"n_heads": 8, "qkv": t, "out": None}),
                     ((), {"out": None, "qkv": t}), ((), {"src": torch.zeros(1), "pages": t})):
        entered.clear()
        assert fn(*args, **kw) == len(args) + len(kw) and entered == [torch.device("cuda", 1)], kw
    entered.clear()
    assert fn(n_heads=8) == 1 and fn(torch.zeros(1), 2) == 2 and not entered


def test_prompt_tables_of_2_30_positions_are_refused():
    """The key blocks of 256 pairs are added up in 32 bits: 2^23 of each would be 2^31."""
    uns = _lib.ERR_UNSUPPORTED
    for ps, most in ((256, 2 ** 22), (16, 2 ** 26)):
        kw = dict(ps=ps, ts=most, ks=ps * 512, vs=ps * 512, wsb=0)
        assert code("nkimoe_paged_prefill_attention", *prefill_args(mp=most, **kw)) == uns
        # one page less is a matter of the workspace alone
        assert code("nkimoe_paged_prefill_attention", *prefill_args(mp=most - 1, **kw)) == _lib.ERR_WORKSPACE


def test_token_ids_on_the_host_are_checked():
    from nki_moe_b200.qwen_stack import _token_ids

    for ok in (torch.tensor([[0, 99]]), torch.tensor([5], dtype=torch.int32), torch.zeros(0, dtype=torch.int64),
               torch.tensor([99], dtype=torch.uint8)):
        assert _token_ids(ok, 100).shape == (ok.numel(),)
    for bad in (torch.tensor([3, 100]), torch.tensor([-1]), torch.tensor([2 ** 40]), torch.rand(2),
                torch.zeros(2, dtype=torch.bool), torch.zeros(1, dtype=torch.complex64)):
        with pytest.raises(ValueError):
            _token_ids(bad, 100)
