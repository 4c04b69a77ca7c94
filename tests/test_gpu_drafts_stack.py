"""Drafted tokens in the decoder stack: steps with trees against HF (bars: see
``test_gpu_stack.py``), generation with drafts and with restricted sampling."""

import math

import pytest
import torch

from tests.test_gpu_paged_stack import hf_logits, ids
from tests.test_gpu_stack import NORM_BAR, _check, tiny_hf

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


def lines(parents):
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


TREES = [[-1, 0, 1, 1, 0, 4, 2], [-1], [-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 6, 6, 3, 1, 0, 14, 15, 16, 17, 18, 19]]


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_logits_after_every_node(pair, window, sinks):
    """A node's logits are those of the text that ends in its path; what is accepted goes on as
    if it had come one by one."""
    hf, st = pair
    prompts = [ids(n, n) for n in (50, 17, 100)]
    cache = st.paged_cache(40, page_size=16, window=window, sinks=sinks)
    seqs = [cache.add() for _ in prompts]
    st.prefill_paged(cache, seqs, prompts)
    texts = [p.clone() for p in prompts]
    for turn in range(3):
        trees = [TREES[(i + turn) % 3] for i in range(3)]
        tokens = [ids(len(t), 10 * turn + i) for i, t in enumerate(trees)]
        logits, step = st.draft_paged(cache, seqs, tokens, trees)
        # every node's own text
        ref, at = [], 0
        for text, tree, tok in zip(texts, trees, tokens):
            for line in lines(tree):
                ref.append(hf_logits(hf, torch.cat([text, tok[line]]), window, sinks)[-1])
        _check(logits, torch.stack(ref))
        # the drawn tokens agree with the last node's path
        sampled = torch.full((logits.shape[0],), 1023, dtype=torch.int64)
        for i, (tree, tok) in enumerate(zip(trees, tokens)):
            line = lines(tree)[-1]
            for a, b in zip(line, line[1:]):
                sampled[at + a] = tok[b]
            texts[i] = torch.cat([texts[i], tok[line]])
            at += len(tree)
        rows = st.accept_paged(cache, step, sampled.cuda())
        assert [len(r) for r in rows] == [len(lines(t)[-1]) for t in trees]
        assert [cache.length(q) for q in seqs] == [len(t) for t in texts]
    got = st.decode_paged(cache, seqs, ids(3, 77))
    ref = [hf_logits(hf, torch.cat([t, ids(3, 77)[i:i + 1]]), window, sinks)[-1] for i, t in enumerate(texts)]
    _check(got, torch.stack(ref))
    st.release_graph()


def test_chains_are_the_default_and_a_step_may_be_taken_back(pair):
    hf, st = pair
    text = ids(60, 3)
    cache = st.paged_cache(20, page_size=16)
    a = cache.add()
    st.prefill_paged(cache, [a], [text[:40]])
    b = cache.fork(a)
    logits, step = st.draft_paged(cache, [b, a], [text[40:50], text[40:41]])
    ref = hf_logits(hf, text)
    _check(logits, torch.cat([ref[40:50], ref[40:41]]))
    cache.take_back([b, a], [40, 40])
    with pytest.raises(ValueError):
        st.accept_paged(cache, step, torch.zeros(11, dtype=torch.int64, device="cuda"))
    logits, step = st.draft_paged(cache, [a, b], [text[40:44], text[40:60]])
    _check(logits, torch.cat([ref[40:44], ref[40:60]]))
    sampled = torch.cat([text[41:45], text[41:60], text[:1]]).cuda()
    rows = st.accept_paged(cache, step, sampled)
    assert rows[0].tolist() == [0, 1, 2, 3] and rows[1].tolist() == list(range(4, 24))
    assert cache.length(a) == 44 and cache.length(b) == 60


def test_pages_may_move_but_not_be_shared_within_a_step(pair):
    hf, st = pair
    text = ids(70, 4)
    cache = st.paged_cache(20, page_size=16)
    hole = cache.add()
    cache.extend([hole], [64])
    seq = cache.add()
    st.prefill_paged(cache, [seq], [text[:40]])
    parents = [-1, 0, 0, 2, 3]
    tokens = torch.stack([text[40], text[0], text[41], text[42], text[43]])
    logits, step = st.draft_paged(cache, [seq], [tokens], [parents])
    cache.free(hole)
    assert cache.compact()
    sampled = torch.stack([text[41], text[0], text[42], text[43], text[44]]).cuda()
    other = cache.fork(seq)
    with pytest.raises(ValueError, match="forked"):
        st.accept_paged(cache, step, sampled)
    cache.free(other)
    rows = st.accept_paged(cache, step, sampled)
    assert rows[0].tolist() == [0, 2, 3, 4] and cache.length(seq) == 44
    logits, step = st.draft_paged(cache, [seq], [text[44:47]])
    rows = st.accept_paged(cache, step, text[45:48].cuda())
    assert rows[0].tolist() == [0, 1, 2] and cache.length(seq) == 47
    with pytest.raises(ValueError):  # it has ended, with all of its nodes
        st.accept_paged(cache, step, text[:3].cuda())
    cache.take_back([seq], [44])
    _check(st.prefill_paged(cache, [seq], [text[44:]]), hf_logits(hf, text)[-1:])


def own_choice(hf, text, tokens):
    """How far each token's HF logit lies below the largest, relative to the largest logit."""
    logits = hf_logits(hf, torch.cat([text, tokens]))[len(text) - 1:-1]
    return (logits.amax(-1) - logits.gather(-1, tokens[:, None])[:, 0]) / logits.abs().amax(-1)


def test_generation_with_drafts_takes_fewer_steps(pair, monkeypatch):
    hf, st = pair
    unit = ids(7, 1)
    prompts = [unit.repeat(6), torch.cat([ids(20, 2), ids(20, 2)]), ids(5, 3)]
    steps = []
    draft = type(st).draft_paged

    def counted(self, cache, seqs, tokens, parents=None):
        steps.append([len(t) for t in tokens])
        return draft(self, cache, seqs, tokens, parents)

    monkeypatch.setattr(type(st), "draft_paged", counted)
    tok, sc = st.generate_paged(prompts, 40, samples=2, top_logprobs=3, page_size=16, drafts=9)
    assert tok.shape == (3, 2, 40) and sc["top_ids"].shape == (3, 2, 40, 3) and sc["logprob"].shape == (3, 2, 40)
    assert torch.equal(tok[:, 0], tok[:, 1]) and torch.equal(sc["top_ids"][..., 0], tok)
    assert max(map(max, steps)) > 1 and max(map(max, steps)) <= 10
    # an untrained model soon repeats itself; each token is the one that HF would choose, to the bar
    assert len(steps) < 39
    for p, t in zip(prompts, tok[:, 0].cpu()):
        assert (own_choice(hf, p, t) <= 2 * NORM_BAR).float().mean() >= 0.9
    assert st._paged is None


def test_drafts_never_ask_for_more_than_there_is(pair):
    _, st = pair
    prompts = [ids(4, 8).repeat(8), ids(4, 9).repeat(3)]
    for pages, size in ((6, 16), (5, 16)):  # 32 + 20 and 12 + 20 positions: four pages and two; one or none to spare
        cache = st.paged_cache(pages + 1, page_size=size, max_seq=64)
        tok, _ = st.generate_paged(prompts, 20, cache=cache, drafts=30)
        assert tok.shape == (2, 1, 20) and cache.free_pages == pages + 1
    one, _ = st.generate_paged(prompts, 1, drafts=5)
    assert one.shape == (2, 1, 1)
    windowed, _ = st.generate_paged(prompts, 50, window=30, sinks=2, page_size=16, drafts=7)
    assert windowed.shape == (2, 1, 50)


def test_restricted_sampling(pair):
    """Samples lie among the tokens that are kept, and the same random numbers give the same text."""
    from nki_moe_b200 import ops

    _, st = pair
    prompts = [ids(20, 6), ids(51, 7)]

    def gen(seed, **kw):
        return st.generate_paged(prompts, 12, samples=3, temperature=1.0, page_size=16, top_logprobs=4,
                                 generator=torch.Generator(device="cuda").manual_seed(seed), **kw)

    for kw in (dict(top_k=4), dict(top_k=4, drafts=6), dict(top_k=4, top_p=0.9, min_p=0.01)):
        a, sc = gen(1, **kw)
        b, _ = gen(1, **kw)
        c, _ = gen(2, **kw)
        assert torch.equal(a, b) and not torch.equal(a, c) and a.shape == (2, 3, 12)
        assert (sc["top_ids"] == a[..., None]).any(-1).all()
    one, _ = gen(3, top_k=1)
    greedy, _ = st.generate_paged(prompts, 12, page_size=16)
    assert torch.equal(one[:, 0], greedy[:, 0])
    logits = torch.randn(5, 1024, device="cuda")
    u = torch.rand(5, dtype=torch.float64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    want, _ = ops.sample_tokens(logits, u, 0.7, 10, 0.8, 0.05)
    assert torch.equal(st._draw(logits, 0.7, 10, 0.8, 0.05, torch.Generator(device="cuda").manual_seed(4)), want)
    st.release_graph()


def test_refusals(pair):
    _, st = pair
    cache = st.paged_cache(8, page_size=16)
    a, b = cache.add(), cache.add()
    st.prefill_paged(cache, [a, b], [ids(5, 1), ids(9, 2)])
    one = ids(1, 1)
    for seqs, tokens, parents in (([a], [], None), ([], [], None), ([a], [ids(0, 1)], None), ([a, a], [one, one], None),
                                  ([a], [ids(65, 1)], None), ([a], [ids(3, 1)], [[-1, 0]]), ([a], [ids(3, 1)], [[-1, 0, 2]]),
                                  ([a], [ids(3, 1)], [[-1, -1, 0]]), ([a], [ids(2, 1)], [[0, 0]]), ([99], [one], None),
                                  ([a], [torch.tensor([1024])], None), ([a], [torch.rand(2)], None)):
        with pytest.raises(ValueError):
            st.draft_paged(cache, seqs, tokens, parents)
        assert cache.length(a) == 5 and cache.length(b) == 9
    with pytest.raises(RuntimeError):
        st.draft_paged(cache, [a, b], [ids(60, 1), ids(60, 2)])
    assert cache.length(a) == 5 and cache.free_pages == 6
    for kw in (dict(top_k=-1), dict(top_p=1.5), dict(min_p=-0.5), dict(drafts=64), dict(drafts=-1),
               dict(temperature=-1.0, top_k=3), dict(temperature=float("nan"), drafts=3)):
        with pytest.raises(ValueError):
            st.generate_paged([ids(4, 1)], 4, **kw)


def test_logits_without_a_distribution_are_refused(pair):
    _, st = pair
    head = st.lm_head
    try:
        st.lm_head = torch.full_like(head, math.nan)
        for kw in (dict(drafts=4), dict(), dict(graph=False)):
            with pytest.raises(RuntimeError, match="distribution"):
                st.generate_paged([ids(9, 1), ids(20, 2)], 3, temperature=1.0, top_k=5, **kw)
    finally:
        st.lm_head = head
        st.release_graph()
    tokens, _ = st.generate_paged([ids(9, 1), ids(20, 2)], 3, temperature=1.0, top_k=10 ** 30)
    assert int(tokens.min()) >= 0
