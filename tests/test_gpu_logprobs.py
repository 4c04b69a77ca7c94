"""Token scores against the formulas in 64 bits.

Bars.  Log probabilities are differences of fp32 numbers up to |d| <= 40: each
rounding is at most 2^-24 * 40 = 2^-18.7, and the sum of V terms, kept per
thread over at most a few hundred and joined pairwise, is off by less than
2^-16 relative, so 2^-15 absolute covers both; the entropy, at most 13, is a
ratio of two such sums (2^-15 * 13 < 2^-11).  Ids are exact.
"""

import pytest
import torch

from nki_moe_b200 import ops

pytestmark = pytest.mark.gpu

LP, ENT = 2 ** -15, 2 ** -11


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def check(logits, tokens, top_n):
    lp, ent, tlp, tid = (t.cpu() for t in ops.token_logprobs(logits, tokens, top_n))
    x = logits.double().cpu()
    ref = torch.log_softmax(x, -1)
    given = ref.gather(-1, tokens.cpu().clamp(min=0)[:, None])[:, 0]
    given = torch.where(tokens.cpu() < 0, torch.zeros_like(given), given)

    def same(a, b, tol):
        a = a.double()
        fin = torch.isfinite(b)
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~fin & ~torch.isnan(b)], b[~fin & ~torch.isnan(b)])
        # relative for values far out: an fp32 result of size |b| rounds by 2^-24 |b|
        assert ((a - b).abs()[fin] <= tol + 2 ** -22 * b.abs()[fin]).all(), float((a - b).abs()[fin].max())

    same(lp, given, LP)
    p = ref.exp()
    same(ent, -(p * torch.where(p > 0, ref, torch.zeros_like(ref))).sum(-1), ENT)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top_n]
    assert torch.equal(tid, ids)
    same(tlp, ref.gather(-1, ids), LP)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,n", [(1, 1, 1), (1, 5, 5), (3, 31, 20), (2, 33, 32), (5, 257, 7), (4, 16384, 20),
                                   (4, 16391, 32), (3, 50257, 0), (8, 151936, 20), (2, 151936, 32), (300, 4099, 5),
                                   (700, 20001, 3), (1, 1000003, 20)])
def test_scores(dtype, T, V, n):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    x = (2.5 * torch.randn(T, V, generator=g, device="cuda")).to(dtype)
    tok = torch.randint(V, (T,), generator=g, device="cuda")
    tok[0] = V - 1
    check(x, tok, n)


@pytest.mark.parametrize("V", [40, 16400, 40001])
def test_equal_logits_come_by_id(V):
    """Constant rows, two values, and a row that climbs: more candidates than a chunk's buffer takes."""
    x = torch.zeros(6, V, device="cuda")
    x[1] = -0.0
    x[1, 1::2] = 0.0
    x[2, ::3] = 1.0
    x[3] = torch.arange(V, device="cuda").float() / V
    x[4] = -torch.arange(V, device="cuda").float() / V
    x[5, V - 5:] = 3.0
    check(x, torch.arange(6, device="cuda"), 20)
    check(x[:, :V // 2 * 2].bfloat16(), torch.arange(6, device="cuda"), 32)


def test_masked_vocabulary_infinities_and_nan():
    g = torch.Generator().manual_seed(3)
    V = 33000
    x = torch.randn(9, V, generator=g)
    low = torch.finfo(torch.float32).min
    x[0, 10:] = -torch.inf          # ten tokens left
    x[1, :] = -torch.inf
    x[1, 17000] = 2.0               # one token left
    x[2, 5:] = low                  # masked with the type's lowest value
    x[3, :] = -torch.inf            # nothing left
    x[4, 20000] = torch.nan
    x[5, 7] = torch.inf
    x[6, :] = low                   # the lowest value everywhere: all alike
    x[7, 3] = 3e38
    x[7, 9] = -3e38
    x[8, :] = -torch.inf
    x[8, 32999] = torch.nan
    tok = torch.tensor([3, 17000, 2, 0, 5, 7, 11, 3, 1])
    lp, ent, tlp, tid = (t.cpu() for t in ops.token_logprobs(x.cuda(), tok.cuda(), 12))
    for r in (3, 4, 5, 8):
        assert torch.isnan(lp[r]) and torch.isnan(ent[r])
    assert tid[4, 0] == 20000 and tid[5, 0] == 7 and tid[8, 0] == 32999
    assert lp[1] == 0 and ent[1] == 0 and tid[1].tolist() == [17000] + list(range(11))
    assert (tlp[1, 1:] == -torch.inf).all()
    rows = [0, 1, 2, 6, 7]
    check(x[rows].cuda(), tok[rows].cuda(), 12)


def test_tokens_not_given_and_out_of_range():
    x = torch.randn(4, 500, device="cuda")
    lp, ent, _, _ = ops.token_logprobs(x, torch.tensor([-1, 500, 499, -100], device="cuda"))
    assert lp[0] == 0 and torch.isnan(lp[1]) and torch.isfinite(lp[2]) and lp[3] == 0 and torch.isfinite(ent).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_at_odd_places(dtype):
    """Rows that start and end anywhere relative to 16 bytes, inside values that must not count."""
    buf = torch.full((6 * 5003 + 9,), 100.0, device="cuda", dtype=dtype)
    for off in range(9):
        x = buf[off:off + 6 * 5003].view(6, 5003)[:, 1:4999]
        keep = buf.clone()
        x.copy_(torch.randn(6, 4998, device="cuda"))
        check(x, torch.tensor([0, 4997, 1, 2, 3, 4], device="cuda"), 5)
        buf.copy_(keep)


def test_calls_on_two_streams_and_in_graphs():
    x = [torch.randn(4, 60000, device="cuda") for _ in range(2)]
    tok = torch.tensor([1, 2, 3, 4], device="cuda")
    want = [ops.token_logprobs(v, tok, 8) for v in x]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = ops.token_logprobs(v, tok, 8)
        graphs.append((g, got))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.token_logprobs(x[0], tok, 8)
    torch.cuda.synchronize()
    for (_, got), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


@pytest.mark.parametrize("dtype,n", [(torch.float32, 20), (torch.bfloat16, 5), (torch.bfloat16, 32)])
def test_orders_within_whole_rows(dtype, n):
    """Rows that one CTA reads in several chunks: rising, falling, few different values,
    all below zero, all of the best in one warp's or one lane's places, the best last."""
    T, V = 600, 25003
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(T, V, generator=g, device="cuda")
    at = torch.arange(V, device="cuda")
    x[0:100] = x[0:100].sort(-1).values
    x[100:200] = x[100:200].sort(-1, descending=True).values
    x[200:300] = (2 * x[200:300]).round()
    x[300:400] = -5 - x[300:400].abs()
    x[400:450] += 20.0 * ((at // 256) % 8 == 3)
    x[450:500] += 20.0 * ((at // 8) % 256 == 77)
    x[500:550, -40:] += 10
    x[550:600] = -torch.inf
    x[550:600, ::911] = 0.5
    check(x.to(dtype), torch.randint(V, (T,), generator=g, device="cuda"), n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 6, 17, 32])
def test_alternatives_of_rows_whose_best_keep_changing(dtype, n):
    """Every chunk of the row holds new best tokens of every warp, so what the warps
    show each other changes all the time."""
    T, V = 640, 40003
    g = torch.Generator(device="cuda").manual_seed(7 + n)
    x = torch.randn(T, V, generator=g, device="cuda") + torch.arange(V, device="cuda") / 1000
    x[::3] = (4 * x[::3]).round() / 4  # and ties among them
    check(x.to(dtype), torch.randint(V, (T,), generator=g, device="cuda"), n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [500, 8192, 20011])
@pytest.mark.parametrize("n", [0, 5])
def test_large_maxima(dtype, V, n):
    """A logit far above the others, of any size that the type holds, with and without
    excluded tokens next to it: all the weight lies on it, or half where there are two.
    Results are fp32: what lies further out than the type reaches, the log probability of a
    token masked with the lowest value under a maximum of 3e38, is -inf, as its rounding is."""
    tops = [1e29, 9e29, 1e31, 2e31, 1e32, 1e36, 1.5e36, 9e36, 1.1e37, 1e38, 3e38]
    x = torch.zeros(4 * len(tops), V, device="cuda")
    for i, m in enumerate(tops):
        x[4 * i:4 * i + 4, V // 3] = m
        x[4 * i + 1, ::7] = -torch.inf
        x[4 * i + 2, V - 2] = m
        x[4 * i + 3, 1::2] = torch.finfo(dtype).min
        x[4 * i:4 * i + 4, V // 3] = m
    x, tok = x.to(dtype), torch.arange(4 * len(tops), device="cuda") % V
    lp, ent, tlp, tid = (t.cpu() for t in ops.token_logprobs(x, tok, n))
    ref = torch.log_softmax(x.double().cpu(), -1)
    p = ref.exp()
    ids = torch.sort(x.cpu().double(), dim=-1, descending=True, stable=True).indices[:, :n]
    assert torch.equal(tid, ids)
    for got, want in ((lp, ref.gather(-1, tok.cpu()[:, None])[:, 0]), (tlp, ref.gather(-1, ids))):
        want = want.float().double()
        far = torch.isinf(want)
        assert torch.equal(got.double()[far], want[far])
        assert ((got.double() - want).abs()[~far] <= LP + 2 ** -22 * want.abs()[~far]).all()
    assert ((ent.double() + (p * torch.where(p > 0, ref, torch.zeros_like(ref))).sum(-1)).abs() <= ENT).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 500, 8192, 20011])
def test_rows_of_the_lowest_values(dtype, V):
    """Rows whose largest logit is the type's lowest finite value, or next to it: the tokens
    that share it are equally likely, excluded ones and places outside the row count for nothing."""
    low = torch.finfo(dtype).min
    x = torch.full((6, V), low, device="cuda", dtype=dtype)
    x[1, ::2] = -torch.inf
    x[2, :] = -torch.inf
    x[2, V - 1] = low
    x[3, 1] = torch.tensor(low, dtype=dtype) * (1 - torch.finfo(dtype).eps)
    x[4] = -1e31
    x[5, 2:4] = -2e30
    for top_n in (0, min(V, 7)):
        check(x, torch.tensor([0, 1, V - 1, 1, 2, 3], device="cuda"), top_n)
