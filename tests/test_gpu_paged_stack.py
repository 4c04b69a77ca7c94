"""The decoder stack on its paged cache, against HF ``Qwen3MoeForCausalLM``
(bars: see ``test_gpu_stack.py``): prompts of different lengths, chunks,
forks, windows, graph and eager steps, scores."""

import pytest
import torch

from tests.test_gpu_stack import NORM_BAR, QUANTILE, _check, tiny_hf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def pair():
    from nki_moe_b200.qwen_stack import Qwen3MoEStack

    hf = tiny_hf()
    return hf, Qwen3MoEStack.from_hf(hf, max_batch=4, max_seq=256)


def ids(n, seed):
    return torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(seed))


def hf_logits(hf, tokens, window=0, sinks=0):
    """All logits of one text; with a window through an explicit mask."""
    mask = None
    if window:
        n = len(tokens)
        p, s = torch.arange(n)[:, None], torch.arange(n)
        see = (s <= p) & ((s > p - window) | (s < sinks))
        mask = torch.zeros(1, 1, n, n).masked_fill(~see, torch.finfo(torch.float32).min)
    with torch.no_grad():
        return hf(tokens[None], attention_mask=mask).logits[0]


@pytest.mark.parametrize("graph", [False, True])
def test_prompts_of_different_lengths_then_steps(pair, graph):
    hf, st = pair
    texts = [ids(n + 6, n) for n in (1, 17, 40, 100, 130)]
    cache = st.paged_cache(40, page_size=16)
    seqs = [cache.add() for _ in texts]
    got = [st.prefill_paged(cache, seqs, [t[:-6] for t in texts])]
    for i in range(6, 0, -1):
        step = torch.stack([t[-i] for t in texts]).cuda()
        got.append(st.decode_paged(cache, seqs, step, graph=graph))
    got = torch.stack(got, 1)
    ref = torch.stack([hf_logits(hf, t)[-7:] for t in texts])
    _check(got.reshape(-1, 1024), ref.reshape(-1, 1024))
    st.release_graph()


def test_a_prompt_in_chunks_equals_the_whole(pair):
    hf, st = pair
    text = ids(150, 3)
    cache = st.paged_cache(20, page_size=32)
    seq = cache.add()
    got = [st.prefill_paged(cache, [seq], [text[a:b]])[0] for a, b in ((0, 1), (1, 33), (33, 100), (100, 150))]
    ref = hf_logits(hf, text)
    _check(torch.stack(got), ref[[0, 32, 99, 149]])


@pytest.mark.parametrize("window,sinks", [(40, 4), (16, 0)])
def test_window_and_first_tokens(pair, window, sinks):
    hf, st = pair
    texts = [ids(n, n) for n in (150, 90)]
    cache = st.paged_cache(30, page_size=16, window=window, sinks=sinks)
    seqs = [cache.add() for _ in texts]
    got = [st.prefill_paged(cache, seqs, [t[:-8] for t in texts])]
    held = 30 - cache.free_pages
    assert held <= 2 * (window // 16 + 3)  # the rest was given back
    for i in range(8, 0, -1):
        got.append(st.decode_paged(cache, seqs, torch.stack([t[-i] for t in texts])))
    got = torch.stack(got, 1)
    ref = torch.stack([hf_logits(hf, t, window, sinks)[-9:] for t in texts])
    _check(got.reshape(-1, 1024), ref.reshape(-1, 1024))
    st.release_graph()


def test_forks_go_their_own_ways_and_compaction_keeps_them(pair):
    hf, st = pair
    prompt, ways = ids(37, 5), [ids(6, 50 + i) for i in range(3)]
    cache = st.paged_cache(40, page_size=16)
    hole = cache.add()
    cache.extend([hole], [64])
    first = cache.add()
    st.prefill_paged(cache, [first], [prompt])
    seqs = [first, cache.fork(first), cache.fork(first)]
    assert cache.free_pages == 40 - 4 - 3
    got = []
    for i in range(6):
        got.append(st.decode_paged(cache, seqs, torch.stack([w[i] for w in ways])))
        if i == 2:
            cache.free(hole)
            assert cache.compact()
    ref = torch.stack([hf_logits(hf, torch.cat([prompt, w]))[-6:] for w in ways])
    _check(torch.stack(got, 1).reshape(-1, 1024), ref.reshape(-1, 1024))
    st.release_graph()


def test_generate_samples_and_scores(pair):
    _, st = pair
    prompts = [ids(20, 6), ids(51, 7)]
    tok, sc = st.generate_paged(prompts, 8, samples=2, top_logprobs=5, page_size=16)
    assert tok.shape == (2, 2, 8) and torch.equal(tok[:, 0], tok[:, 1])  # greedy: the samples are alike
    assert torch.equal(sc["top_ids"][..., 0], tok) and torch.equal(sc["top_logprobs"][..., 0], sc["logprob"])
    assert sc["top_ids"].shape == (2, 2, 8, 5) and (sc["entropy"] >= 0).all()
    eager, none = st.generate_paged(prompts, 8, page_size=16, graph=False)
    assert none is None and torch.equal(eager[:, 0], tok[:, 0])

    def sampled(seed):
        return st.generate_paged(prompts, 8, samples=3, temperature=1.0,
                                 generator=torch.Generator(device="cuda").manual_seed(seed))[0]

    a, b, c = sampled(1), sampled(1), sampled(2)
    assert torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(a[:, 0], a[:, 1])
    cache = st.paged_cache(8, page_size=16)
    st.generate_paged([prompts[0]], 4, samples=2, cache=cache)
    assert cache.free_pages == 8
    with pytest.raises(RuntimeError):
        st.generate_paged(prompts * 2, 4, samples=2, cache=cache)
    assert cache.free_pages == 8
    st.release_graph()


def test_score_of_given_texts(pair):
    hf, st = pair
    texts = [ids(n, 60 + n) for n in (1, 2, 70, 120)]
    got = st.score(texts, top_n=3, page_size=16, chunk=50)
    for text, (lp, ent, tlp, tid) in zip(texts, got):
        n = len(text) - 1
        assert lp.shape == ent.shape == (n,) and tlp.shape == tid.shape == (n, 3)
        if not n:
            continue
        logits = hf_logits(hf, text)[:-1]
        ref = torch.log_softmax(logits.double(), -1).gather(-1, text[1:, None])[:, 0]
        # logits are within NORM_BAR of the largest at 95% of the positions, a
        # log probability within twice that
        bar = 2 * NORM_BAR * logits.abs().amax(-1)
        assert ((lp.cpu() - ref).abs() <= bar).float().mean() >= QUANTILE or n < 20


def test_refusals(pair):
    _, st = pair
    cache = st.paged_cache(4, page_size=16)
    a, b = cache.add(), cache.add()
    for seqs, prompts in (([a], []), ([], []), ([a], [ids(0, 1)]), ([a, a], [ids(3, 1)] * 2), ([77], [ids(3, 1)])):
        with pytest.raises(ValueError):
            st.prefill_paged(cache, seqs, prompts)
    st.prefill_paged(cache, [a, b], [ids(5, 1), ids(9, 2)])
    with pytest.raises(ValueError):
        st.decode_paged(cache, [a, b], torch.tensor([1]))
    with pytest.raises(ValueError):
        st.decode_paged(cache, [a, a], torch.tensor([1, 2]))
    with pytest.raises(RuntimeError):
        st.prefill_paged(cache, [a], [ids(60, 3)])
    assert cache.length(a) == 5 and cache.free_pages == 2


def test_generation_keeps_no_cache_of_its_own(pair):
    """The captured step of a cache that nobody else can reach ends with the call; a
    given cache keeps its step, its pages come back, and its window is not overruled."""
    _, st = pair
    prompts = [ids(20, 1), ids(33, 2)]
    st.release_graph()
    mine, _ = st.generate_paged(prompts, 4, page_size=16)
    assert st._paged is None
    cache = st.paged_cache(12, page_size=16, window=64, sinks=2)
    given, _ = st.generate_paged(prompts, 4, cache=cache)  # nothing is outside the window yet
    assert st._paged["cache"] is cache and cache.free_pages == 12
    assert torch.equal(mine, given)
    again, _ = st.generate_paged(prompts, 4, cache=cache, window=64, sinks=2)
    assert torch.equal(mine, again)
    for kw in (dict(window=32), dict(window=64, sinks=4), dict(sinks=2)):
        with pytest.raises(ValueError):
            st.generate_paged(prompts, 4, cache=cache, **kw)
    assert cache.free_pages == 12
    for size in (0, -16, 24):
        with pytest.raises(ValueError):
            st.generate_paged(prompts, 4, page_size=size)
        with pytest.raises(ValueError):
            st.score(prompts, page_size=size)
    for none in ([], [ids(0, 1)]):
        with pytest.raises(ValueError):
            st.generate_paged(none, 4)
        with pytest.raises(ValueError):
            st.score(none)
    with pytest.raises(ValueError):
        st.score(prompts, chunk=-1)
    st.release_graph()


class _Counted:
    """An expert block in the place of a layer's exchange: what runs on the device is counted there."""

    def __init__(self, lyr, top_k):
        from nki_moe_b200 import ops

        self.count = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.block = lambda x: ops.moe_block(x, lyr.router_w, lyr.experts, top_k, router_w_split=lyr.router_split)

    def __call__(self, x):
        self.count.add_(1)
        return self.block(x)

    def close(self):
        pass


def test_a_call_runs_each_exchange_once():
    """Ranks of an expert-parallel stack stay in step whatever their batches do: a call runs
    each layer's exchange once, whether it captures a step, replays one or neither."""
    from nki_moe_b200.qwen_stack import Qwen3MoEStack

    st = Qwen3MoEStack.from_hf(tiny_hf(), max_batch=4, max_seq=256)
    for lyr in st.layers:
        lyr.ep, lyr.ep_decode = _Counted(lyr, st.cfg.num_experts_per_tok), _Counted(lyr, st.cfg.num_experts_per_tok)
    cache = st.paged_cache(20, page_size=16)
    seqs = [cache.add() for _ in range(4)]
    calls = 0
    st.prefill_paged(cache, seqs, [ids(5, 1)] * 4)
    for B, graph in ((4, True), (4, True), (3, True), (4, True), (2, False), (3, True), (1, True), (1, True)):
        st.decode_paged(cache, seqs[:B], ids(B, calls), graph=graph)
        calls += 1
        for lyr in st.layers:
            assert int(lyr.ep_decode.count) == calls and int(lyr.ep.count) == 1
    st.close()


def test_steps_of_several_batch_sizes_and_caches_are_kept(pair):
    """A batch that grows and shrinks replays the steps that it captured before, with the
    logits of steps that were never captured."""
    _, st = pair
    st.release_graph()
    caches = [st.paged_cache(40, page_size=16) for _ in range(4)]  # 0, 1 with graphs; 2, 3 without
    prompts = [ids(n, 80 + n) for n in (5, 20, 33)]
    seqs = []
    for c in caches:
        seqs.append([c.add() for _ in prompts])
        st.prefill_paged(c, seqs[-1], prompts)
    graphs = {}
    for i, (c, B) in enumerate(((0, 2), (0, 3), (1, 2), (0, 2), (1, 3), (0, 3), (0, 1), (1, 2), (0, 2), (1, 3), (0, 1))):
        tok = ids(B, i)
        got = st.decode_paged(caches[c], seqs[c][:B], tok)
        want = st.decode_paged(caches[c + 2], seqs[c + 2][:B], tok, graph=False)
        assert torch.equal(got, want), (c, B)
        assert graphs.setdefault((c, B), st._paged["graph"]) is st._paged["graph"]
    assert len({id(g) for g in graphs.values()}) == len(graphs) == 5
    st.release_graph()
    assert st._paged is None


def test_the_steps_used_last_are_kept_and_those_of_a_cache_end_with_it(pair, monkeypatch):
    _, st = pair
    st.release_graph()
    monkeypatch.setattr(type(st), "PAGED_STEPS", 2)
    cache = st.paged_cache(20, page_size=16)
    seqs = [cache.add() for _ in range(3)]
    st.prefill_paged(cache, seqs, [ids(4, i) for i in range(3)])
    for B, kept in ((1, [1]), (2, [1, 2]), (1, [2, 1]), (3, [1, 3]), (3, [1, 3]), (2, [3, 2])):
        st.decode_paged(cache, seqs[:B], ids(B, B))
        assert list(st._paged_steps[cache]) == kept
    del cache
    assert len(st._paged_steps) == 0 and st._paged is None


def test_two_caches_on_two_streams(pair):
    _, st = pair
    st.release_graph()
    prompts = [ids(n, 90 + n) for n in (30, 9)]

    def start(c):
        seqs = [c.add() for _ in prompts]
        st.prefill_paged(c, seqs, prompts)
        return seqs

    caches = [st.paged_cache(20, page_size=16) for _ in range(2)]
    seqs = [start(c) for c in caches]
    toks = [ids(2, i).cuda() for i in range(24)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i, tok in enumerate(toks):
        with torch.cuda.stream(streams[i % 2]):
            got.append(st.decode_paged(caches[i % 2], seqs[i % 2], tok))
    torch.cuda.synchronize()
    for k in range(2):
        cache = st.paged_cache(20, page_size=16)
        mine = start(cache)
        for i in range(k, 24, 2):
            assert torch.equal(got[i], st.decode_paged(cache, mine, toks[i], graph=False)), i
    st.release_graph()


def test_captured_steps_leave_nothing_behind(pair):
    """What a captured step held goes with it; what it had reported does not."""
    import gc

    from nki_moe_b200 import ops
    from nki_moe_b200._lib import NKIMoEError

    _, st = pair
    st.release_graph()
    ops.release_captured_workspaces()
    prompts = [ids(20, 1), ids(33, 2)]

    def use():
        st.generate_paged(prompts, 3, page_size=16)
        gc.collect()  # what other tests left in cycles
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.memory_allocated(), torch.cuda.memory_reserved()

    for _ in range(3):
        use()
    before = use()
    for _ in range(4):
        assert use() == before
    assert not [k for k in ops._paged_ws if k[2]]
    ops.read_paged_status()
    cache = st.paged_cache(8, page_size=16)
    seq = cache.add()
    st.prefill_paged(cache, [seq], [prompts[1]])
    st.decode_paged(cache, [seq], ids(1, 1))
    st.decode_paged(cache, [seq], ids(1, 2))
    page, cache._seqs[seq].pages[1] = cache._seqs[seq].pages[1], 10 ** 6  # no such page
    st.decode_paged(cache, [seq], ids(1, 3))
    cache._seqs[seq].pages[1] = page
    st.decode_paged(cache, [seq], ids(1, 4))  # a good one after it
    st.release_graph()
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    ops.read_paged_status()


def test_a_call_that_fails_leaves_the_lengths(pair, monkeypatch):
    """Nothing counts as held that was not stored: a prompt or a step that fails on the way
    can be given again."""
    hf, st = pair
    text = ids(60, 9)
    cache = st.paged_cache(12, page_size=16)
    seq = cache.add()
    st.prefill_paged(cache, [seq], [text[:20]])
    other = cache.fork(seq)
    free = cache.free_pages

    def fails(*a, **kw):
        raise RuntimeError("out of memory")

    for name in ("_layers", "_paged_body"):
        with monkeypatch.context() as m:
            m.setattr(st, name, fails)
            for graph in (False, True):
                with pytest.raises(RuntimeError, match="out of memory"):
                    if name == "_layers":
                        st.prefill_paged(cache, [seq, other], [text[20:57], text[20:30]])
                    st.decode_paged(cache, [other, seq], text[20:22], graph=graph)
    for bad in (torch.rand(3), torch.zeros(3, dtype=torch.bool)):
        with pytest.raises(ValueError):
            st.prefill_paged(cache, [seq], [bad])
        for graph in (False, True):
            with pytest.raises(ValueError):
                st.decode_paged(cache, [seq], bad[:1], graph=graph)
    assert cache.length(seq) == cache.length(other) == 20 and cache.free_pages >= free - 1  # a copied page may stay
    got = [st.prefill_paged(cache, [seq], [text[20:57]])[0]] + [st.decode_paged(cache, [seq], text[i:i + 1])[0]
                                                                for i in range(57, 60)]
    _check(torch.stack(got), hf_logits(hf, text)[56:60])
    st.release_graph()


def test_a_step_of_no_sequences(pair):
    _, st = pair
    cache = st.paged_cache(4, page_size=16)
    for graph in (False, True, True):
        assert st.decode_paged(cache, [], ids(0, 1), graph=graph).shape == (0, 1024)
    assert cache.free_pages == 4
    st.release_graph()
