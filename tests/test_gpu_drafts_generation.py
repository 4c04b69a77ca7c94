"""Generation with drafts and with restricted sampling against generation without
(bars: see ``test_gpu_stack.py``)."""

import math

import pytest
import torch

from tests.test_gpu_paged_stack import hf_logits, ids
from tests.test_gpu_stack import NORM_BAR, tiny_hf

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


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("kw", [dict(drafts=4), dict(top_k=5), dict(top_p=0.9, graph=False), dict(min_p=0.1, drafts=2),
                                dict(drafts=3, top_logprobs=2)])
def test_logits_without_a_distribution_are_refused_greedy_too(pair, kw, value, temperature):
    _, st = pair
    head = st.lm_head
    cache = st.paged_cache(16, page_size=16)
    try:
        st.lm_head = head.clone()
        st.lm_head[7] = value  # one logit of every row
        with pytest.raises(RuntimeError, match="distribution"):
            st.generate_paged([ids(9, 1), ids(20, 2)], 3, temperature=temperature, cache=cache, **kw)
        assert cache.free_pages == 16
    finally:
        st.lm_head = head
        st.release_graph()
    tokens, _ = st.generate_paged([ids(9, 1), ids(20, 2)], 3, temperature=temperature, **kw)
    assert 0 <= int(tokens.min()) and int(tokens.max()) < 1024


def test_greedy_draws_name_the_first_of_equal_logits(pair):
    _, st = pair
    x = torch.zeros(5, 1024, device="cuda", dtype=torch.bfloat16)
    x[1, 300:600] = 2.0
    x[2] = -math.inf
    x[3, 9] = math.nan
    x[4, 11:] = -math.inf
    assert st._draw(x, 0.0, 0, 1.0, 0.0, None).tolist() == [0, 300, -1, -1, 0]


def test_a_step_that_others_have_overtaken_is_refused(pair):
    """Its nodes' rows are not in the cache any more, or not in this one."""
    _, st = pair
    text = ids(60, 3)
    cache, other = (st.paged_cache(20, page_size=16) for _ in range(2))
    a, b = cache.add(), other.add()
    for c, q in ((cache, a), (other, b)):
        st.prefill_paged(c, [q], [text[:40]])
    assert a == b
    sampled = text[41:46].cuda()
    _, old = st.draft_paged(cache, [a], [ids(5, 1)])
    st.draft_paged(other, [b], [text[40:45]])
    with pytest.raises(ValueError, match="cache"):
        st.accept_paged(other, old, sampled)
    cache.take_back([a], [40])
    _, new = st.draft_paged(cache, [a], [text[40:45]])  # as many nodes
    with pytest.raises(ValueError, match="left"):
        st.accept_paged(cache, old, sampled)
    rows = st.accept_paged(cache, new, sampled)
    assert rows[0].tolist() == [0, 1, 2, 3, 4] and cache.length(a) == 45
    # ended, put back, and grown to the same length by other calls
    _, old = st.draft_paged(cache, [a], [text[45:48]])
    cache.take_back([a], [45])
    st.prefill_paged(cache, [a], [text[45:48]])
    with pytest.raises(ValueError, match="left"):
        st.accept_paged(cache, old, text[46:49].cuda())
    assert cache.length(a) == 48
    # a call behind its nodes that was put back does not touch them
    _, step = st.draft_paged(cache, [a], [text[48:51]])
    st.decode_paged(cache, [a], text[:1], graph=False)
    with pytest.raises(ValueError, match="left"):
        st.accept_paged(cache, step, text[49:52].cuda())
    cache.take_back([a], [51])
    assert st.accept_paged(cache, step, text[49:52].cuda())[0].tolist() == [0, 1, 2] and cache.length(a) == 51


@pytest.fixture(scope="module")
def smooth():
    """A model without a choice of experts (all of them are used), so that no position leaves the bar
    because another one was chosen, whose texts run in rounds now and then, so that drafts come true."""
    from nki_moe_b200.qwen_stack import Qwen3MoEStack

    hf = tiny_hf()
    hf.config.num_experts_per_tok = hf.config.num_experts
    with torch.no_grad():
        for lyr in hf.model.layers:
            lyr.mlp.gate.top_k = hf.config.num_experts
        t = torch.arange(1024)
        w = hf.lm_head.weight.clone()
        w[(t // 7 * 7 + (t % 7 + 1) % 7).clamp(max=1023)] += 0.3 * hf.model.embed_tokens.weight
        hf.lm_head.weight.copy_(w.bfloat16().float())
    return hf, Qwen3MoEStack.from_hf(hf, max_batch=4, max_seq=256)


def counted(monkeypatch, st):
    """The trees' sizes of every step with drafts."""
    steps, draft = [], type(st).draft_paged

    def call(self, cache, seqs, tokens, parents=None):
        steps.append([len(t) for t in tokens])
        return draft(self, cache, seqs, tokens, parents)

    monkeypatch.setattr(type(st), "draft_paged", call)
    return steps


PROMPTS = [ids(7, 1).repeat(6), torch.cat([ids(20, 2), ids(20, 2)]), ids(5, 3)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_greedy_generation_with_drafts_against_generation_without(smooth, monkeypatch, window, sinks):
    """A logit is within e = NORM_BAR of the row's largest of HF's, so a token that is chosen lies at most
    2 e below HF's largest; where HF's two largest are further apart than that, it is HF's own.  Log
    probabilities are within 2 e; an entropy, whose derivative by a logit is -p (log p + H), within e
    times the deviation of log p, which over such a change grows by 2 e and a factor of exp(e)."""
    hf, st = smooth
    kw = dict(samples=2, top_logprobs=2, page_size=16, window=window, sinks=sinks)
    plain, _ = st.generate_paged(PROMPTS, 40, **kw)
    steps = counted(monkeypatch, st)
    drafted, sc = st.generate_paged(PROMPTS, 40, drafts=9, **kw)
    assert len(steps) < 39 and max(map(max, steps)) > 1  # drafts were made, and some came true
    sure = 0
    for i, p in enumerate(PROMPTS):
        for s in range(2):
            for tokens in (drafted[i, s].cpu(), plain[i, s].cpu()):
                logits = hf_logits(hf, torch.cat([p, tokens]), window, sinks)[len(p) - 1:-1].double()
                big = logits.abs().amax(-1)
                top = logits.topk(2, -1).values
                own = logits.gather(-1, tokens[:, None])[:, 0]
                assert ((top[:, 0] - own) <= 2 * NORM_BAR * big).all()
                clear = (top[:, 0] - top[:, 1]) > 2 * NORM_BAR * big
                assert torch.equal(tokens[clear], logits.argmax(-1)[clear])
                sure += int(clear.sum())
            differ = (drafted[i, s] != plain[i, s]).nonzero()
            if len(differ):
                logits = hf_logits(hf, torch.cat([p, plain[i, s].cpu()]), window, sinks)[len(p) - 1 + int(differ[0])]
                top = logits.topk(2).values
                assert top[0] - top[1] <= 2 * NORM_BAR * logits.abs().max()
            tokens = drafted[i, s].cpu()
            logits = hf_logits(hf, torch.cat([p, tokens]), window, sinks)[len(p) - 1:-1].double()
            logp = torch.log_softmax(logits, -1)
            e = NORM_BAR * logits.abs().amax(-1)
            assert ((sc["logprob"][i, s].cpu() - logp.gather(-1, tokens[:, None])[:, 0]).abs() <= 2 * e).all()
            entropy = -(logp.exp() * logp).sum(-1)
            spread = (logp.exp() * (logp + entropy[:, None]) ** 2).sum(-1).sqrt()
            assert ((sc["entropy"][i, s].cpu() - entropy).abs() <= e * e.exp() * (spread + 2 * e)).all()
            assert torch.equal(sc["top_ids"][i, s, :, 0].cpu(), tokens)
    assert sure > 100  # of 240 positions of each
    st.release_graph()


def test_drafted_draws_follow_the_distribution(smooth, monkeypatch):
    """Of 3600 draws as many are the r-th most likely token as their own rows' probabilities add up to, to
    five standard deviations; the rows are what the scores show, restricted to the first four."""
    _, st = smooth
    steps = counted(monkeypatch, st)
    tokens, sc = st.generate_paged(PROMPTS, 12, samples=100, temperature=0.7, top_k=4, top_logprobs=4, page_size=16,
                                   drafts=5, generator=torch.Generator(device="cuda").manual_seed(9))
    assert len(steps) >= 4 and sum(map(sum, steps)) > 1.5 * sum(map(len, steps))
    p = torch.softmax(sc["top_logprobs"].double() / 0.7, -1)
    hit = (sc["top_ids"] == tokens[..., None]).double()
    assert (hit.sum(-1) == 1).all()
    for position in (slice(0, 12), slice(1, 2), slice(11, 12)):
        off = (hit - p)[:, :, position].sum((0, 1, 2))
        dev = (p * (1 - p))[:, :, position].sum((0, 1, 2)).sqrt()
        assert (off.abs() <= 5 * dev).all(), (off, dev)
