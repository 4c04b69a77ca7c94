"""Generation with drafts and with restricted sampling against generation without
(bars: see ``test_gpu_stack.py``)."""

import math

import pytest
import torch

from tests.test_gpu_paged_stack import ids
from tests.test_gpu_stack import tiny_hf

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
