"""Sampling on the GPU against its definition in 64 bits.

Tokens have to be equal: the weights that a draw adds up are whole numbers of 2^-44 of
the largest, each off by 2^-45 at most, whose errors in a sum of V are V / 2 of them at
the very most and the square root of V in earnest (2^-36 for 2^18); histograms hold weights to 2^-32 each; and
no random number here lies nearer to a border than 2^-31 of the sum (checked:
``margin``).  A log probability is one rounding to fp32 (2^-24 of its value) of the
weight's logarithm less that of the sum, which is off by V 2^-45 at most.
"""

import math

import pytest
import torch

from nki_moe_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def drawn(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """Token, log probability, and how near a border a decision was (relative to the sum) for one row."""
    x = x.double()
    if torch.isnan(x).any() or not math.isfinite(float(x.max())) or not t >= 0:
        return -1, math.nan, 1.0
    first = int((x == x.max()).nonzero()[0])
    if t == 0 or k == 1:
        return first, 0.0, 1.0
    order = torch.sort(x, descending=True, stable=True).indices
    order = order[x[order] > -math.inf]
    if k > 0:
        order = order[:k]
    w = ((x[order] - x.max()) / t).exp()
    margin, n = 1.0, len(order)
    if p < 1:
        upto = w.cumsum(0)
        n = min(int((upto < p * upto[-1]).sum()) + 1, len(order))
        margin = float((upto[w > 0] - p * upto[-1]).abs().min() / upto[-1]) if p > 0 else 1.0
    keep = torch.zeros_like(x, dtype=torch.bool)
    keep[order[:n][w[:n] >= min(max(m, 0.0), 1.0)]] = True
    if 0 < m < 1:
        margin = min(margin, float((w - m).abs().min()))
    full = torch.where(keep, ((x - x.max()) / t).exp(), torch.zeros_like(x))
    upto = full.cumsum(0)
    over = (upto > u * upto[-1]) & (full > 0)
    token = int(over.nonzero()[0]) if over.any() else int((full > 0).nonzero()[-1])
    if 0 < u < 1:
        margin = min(margin, float((upto[full > 0] - u * upto[-1]).abs().min() / upto[-1]))
    return token, float((full[token] / upto[-1]).log()), margin


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0, exact_margin=True):
    rows = logits.shape[0]
    dev = [v.cuda() if isinstance(v, torch.Tensor) else v for v in (t, k, p, m)]
    token, lp = ops.sample_tokens(logits.cuda() if not logits.is_cuda else logits, u.cuda(), *dev)
    token, lp = token.cpu(), lp.cpu()
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for i in range(rows):
        want, want_lp, margin = drawn(logits[i].cpu(), u[i].item(), at(t, i), at(k, i), at(p, i), at(m, i))
        if exact_margin:
            assert margin > 2 ** -31, "choose another random number: this one lies on a border"
        assert int(token[i]) == want, f"row {i}: {int(token[i])}, not {want}"
        if math.isnan(want_lp):
            assert math.isnan(float(lp[i]))
        else:
            assert abs(float(lp[i]) - want_lp) <= 2 ** -24 * abs(want_lp) + logits.shape[1] * 2 ** -45 + 1e-12
    return token


def logits_of(rows, vocab, seed, dtype=torch.bfloat16, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    x.scatter_add_(1, torch.randint(vocab, (rows, 8), generator=g), 8 * torch.rand(rows, 8, generator=g))
    return x.to(dtype), torch.rand(rows, generator=g, dtype=torch.float64)


SETTINGS = [dict(), dict(k=5), dict(p=0.9), dict(m=0.05), dict(t=0.6, k=20, p=0.95), dict(t=1.5, p=0.99, m=0.01),
            dict(t=0.0), dict(k=1), dict(k=700, p=0.5, m=0.001), dict(t=0.01), dict(t=30.0, p=0.7), dict(p=0.0),
            dict(m=1.0), dict(k=10 ** 9)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 100, 513, 4099, 50257])
def test_sizes_and_settings(vocab, dtype):
    for i, s in enumerate(SETTINGS):
        x, u = logits_of(3, vocab, 100 * vocab + i, dtype)
        check(x, u, **s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [151936, 262144])
@pytest.mark.parametrize("s", [dict(), dict(t=0.6, k=20, p=0.95), dict(p=0.9), dict(t=1.2, k=30000, p=0.8)])
def test_large_vocabularies(vocab, dtype, s):
    x, u = logits_of(3, vocab, vocab + len(s), dtype)
    check(x, u, **s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(160, 151936), (40, 200003), (200, 47105), (90, 94209)])
def test_rows_enough_for_wide_slices(rows, vocab, dtype):
    """With many rows fewer CTAs share one, so that a slice of it is as long as it gets."""
    x, u = logits_of(rows, vocab, rows, dtype)
    x, u = x.cuda(), u.cuda()
    for s in (dict(temperature=0.8, top_p=0.9), dict(top_k=40)):
        tok, _ = ops.sample_tokens(x, u, **s)
        for i in range(0, rows, 13):
            want = drawn(x[i].cpu(), u[i].item(), s.get("temperature", 1.0), s.get("top_k", 0), s.get("top_p", 1.0))
            assert int(tok[i]) == want[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(300, 50257), (310, 1027), (120, 151937)])
def test_rows_that_keep_few_or_many(rows, vocab, dtype):
    """Few kept logits of a warp's vectors are weighed together, many one by one; both in one row."""
    x, u = logits_of(rows, vocab, 3 * rows, dtype)
    x[::3, vocab // 2:vocab // 2 + 700] = x[::3].float().amax(1, keepdim=True).to(dtype) - 1.5
    x[1::3] *= 0.25
    x, u = x.cuda(), u.cuda()
    for s in (dict(min_p=0.05), dict(min_p=1e-5, temperature=1.5), dict(top_k=900, min_p=0.01), dict(top_p=0.4)):
        tok, lp = ops.sample_tokens(x, u, **s)
        for i in [*range(0, rows, 23), rows - 1]:
            want, want_lp, margin = drawn(x[i].cpu(), u[i].item(), s.get("temperature", 1.0), s.get("top_k", 0),
                                          s.get("top_p", 1.0), s.get("min_p", 0.0))
            if margin > 2 ** -31:
                assert int(tok[i]) == want, (s, i)
                assert abs(float(lp[i]) - want_lp) <= 2 ** -24 * abs(want_lp) + vocab * 2 ** -45 + 1e-12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("values", [[0.0], [1.5, -0.25], [3.0, 2.984375, -40.0]])
@pytest.mark.parametrize("s", [dict(), dict(k=777), dict(k=70001), dict(p=0.31), dict(k=9000, p=0.77), dict(t=0.2, p=0.999)])
def test_equal_logits_go_by_id(values, dtype, s):
    """More equal logits than one sort takes: the border is found by id."""
    g = torch.Generator().manual_seed(len(values))
    x = torch.tensor(values)[torch.randint(len(values), (2, 100003), generator=g)].to(dtype)
    check(x, torch.tensor([0.318309886, 0.9990234], dtype=torch.float64), exact_margin=False, **s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [151936, 262144])
def test_equal_logits_of_whole_rows(vocab, dtype):
    """A CTA adds up a whole row's weights in one bin: 2^18 of 2^31 units each."""
    x = torch.full((1, vocab), 0.75, dtype=dtype, device="cuda").expand(150, -1)
    u = torch.full((150,), 0.318309886, dtype=torch.float64, device="cuda")
    near = (torch.arange(vocab) % 3 * 2.0 ** -100).to(dtype)[None].cuda().expand(150, -1)
    for logits, t, k, p in ((x, 1.0, 0, 0.9), (x, 1e30, 0, 0.4), (x, math.inf, 150001, 0.7), (near, 2.0, 0, 0.45)):
        tok, lp = ops.sample_tokens(logits, u, torch.full((150,), t, device="cuda"), k, p)
        want, want_lp, margin = drawn(logits[0].cpu(), u[0].item(), t, k, p)
        assert margin > 2 ** -31
        assert (tok == want).all()
        assert (lp.double() - want_lp).abs().max() <= 2 ** -24 * abs(want_lp) + vocab * 2 ** -45 + 1e-12


def test_the_smallest_temperatures():
    x, u = logits_of(3, 5003, 23)
    for t in (5e-324, 1e-310, 1e-200):
        check(x, u, t)
        check(x.float(), u, t, 40, 0.9)


def test_signed_zeros_are_equal():
    x = torch.full((1, 40), -0.0)
    x[0, ::2] = 0.0
    for k in (3, 8):
        check(x, torch.tensor([0.55], dtype=torch.float64), k=k)
        check(x.bfloat16(), torch.tensor([0.55], dtype=torch.float64), k=k)


def test_bins_of_far_and_near_values():
    """Logits in a narrow band (one bin of distances, split by their values), and far apart."""
    g = torch.Generator().manual_seed(5)
    near = 7 + 1e-5 * torch.rand(2, 30000, generator=g)
    far = -300 * torch.rand(2, 30000, generator=g)
    far[:, 17] = 5.0
    for x in (near, far, near.bfloat16(), far.bfloat16()):
        for s in (dict(k=9000), dict(p=0.43), dict(k=20000, p=0.6), dict(t=50.0, p=0.9), dict(t=1e4, k=12345)):
            check(x, torch.tensor([0.123456, 0.7654321], dtype=torch.float64), exact_margin=False, **s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_and_broken_rows(dtype):
    x, u = logits_of(9, 3001, 11, dtype)
    x[0, :3000] = -math.inf  # one token left
    x[1] = -math.inf
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = torch.finfo(dtype).min
    x[5] = torch.finfo(dtype).min
    x[5, 2999] = torch.finfo(dtype).max
    x[6, ::2] = -math.inf
    x[7, 1:] = -math.inf
    x[8, 100:] = torch.finfo(dtype).min
    for s in (dict(), dict(k=50), dict(p=0.8), dict(t=0.0), dict(k=2000, p=0.9, m=0.1), dict(k=1)):
        tok = check(x, u, exact_margin=False, **s)
        assert tok[0] == 3000 and tok[1] == tok[2] == tok[3] == -1


def test_rows_whose_sample_misses_what_matters():
    """Whole rows are counted with a window that a sample of them suggests: largest and smallest
    logits far outside of it, all zeros but a few, all tiny, many near zero."""
    rows, vocab = 150, 20011
    x, u = logits_of(rows, vocab, 21)
    x[0:30, 777] = 300.0
    x[30:60, 15001] = -3000.0
    x[60:90] *= 2.0 ** -60
    x[90:100] = 0.0
    x[90:100, ::100] = torch.randn(10, 201, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[100:110, 1::2] *= 2.0 ** -20
    x[110:120] = -x[110:120].abs() - 4
    x[120:130, 5] = -0.0
    x[130:140] = torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0).bfloat16()
    x, u = x.cuda(), u.cuda()
    for s in (dict(temperature=0.9, top_p=0.9), dict(top_k=3000), dict(temperature=200.0, top_p=0.6, top_k=15000),
              dict(temperature=3.0, top_p=0.999), dict(top_k=7, top_p=0.5)):
        tok, lp = ops.sample_tokens(x, u, **s)
        for i in [*range(0, rows, 6), 90, 91, 130, 131]:
            want, want_lp, margin = drawn(x[i].cpu(), u[i].item(), s.get("temperature", 1.0), s.get("top_k", 0),
                                          s.get("top_p", 1.0))
            if margin > 2 ** -31:
                assert int(tok[i]) == want, (s, i)
                assert abs(float(lp[i]) - want_lp) <= 2 ** -24 * abs(want_lp) + vocab * 2 ** -45 + 1e-12


def test_settings_per_row():
    g = torch.Generator().manual_seed(3)
    x, u = logits_of(64, 5003, 12)
    pick = lambda v, dt: torch.tensor(v, dtype=dt)[torch.randint(len(v), (64,), generator=g)]  # noqa: E731
    t = pick([0.0, 0.3, 1.0, 2.0, math.inf, -1.0, math.nan], torch.float32)
    k = pick([-3, 0, 1, 2, 40, 5003, 99999], torch.int32)
    p = pick([0.0, 0.5, 0.95, 1.0, 7.0], torch.float32)
    m = pick([-1.0, 0.0, 0.1, 1.0, 3.0], torch.float32)
    check(x, u, t, k, p, m, exact_margin=False)
    check(x.float(), u.float(), 0.7, k, 0.9, m)
    check(x, u, t, 0, p, 0.0, exact_margin=False)


def test_ends_of_the_unit_interval():
    x, _ = logits_of(4, 20011, 13)
    x[:, :5] = -math.inf
    x[:, -3:] = -math.inf
    u = torch.tensor([0.0, math.nextafter(1.0, 0.0), 0.0, math.nextafter(1.0, 0.0)], dtype=torch.float64)
    # the whole sum is a border too, 2^-53 from the last of these: the last id's own weight is the room there is
    assert check(x, u, exact_margin=False)[0] == 5
    check(x, u, k=30, exact_margin=False)
    check(x, u, p=0.6, exact_margin=False)
    tok, _ = ops.sample_tokens(x.cuda(), torch.tensor([-1.0, 1.0, 2.0, math.nan]).cuda(), 1.0, 3)
    for i, want in enumerate((0, 1, 1, 1)):  # outside of it: the first or the last kept id
        kept = torch.sort(torch.sort(x[i].float(), descending=True, stable=True).indices[:3]).values
        assert int(tok[i]) == int(kept[-want])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_at_any_stride(dtype):
    x, u = logits_of(5, 9001, 14, dtype)
    wide = torch.full((5, 9100), math.nan, dtype=dtype, device="cuda")
    for off in (0, 1, 3, 7, 8):
        view = wide[:, off:off + 9001]
        view.copy_(x)
        check(view, u, k=100, p=0.9)
        check(view, u)
        wide.fill_(math.nan)
    same = x[:1].cuda().expand(5, -1)  # one row for all
    check(same, u, p=0.8)


def test_many_rows_are_deterministic_and_each_on_its_own():
    x, u = logits_of(700, 6007, 15)
    for s in (dict(p=0.9), dict(k=20, p=0.95), dict()):
        a = check(x, u, **s)
        for _ in range(3):
            b, _ = ops.sample_tokens(x.cuda(), u.cuda(), s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0))
            assert torch.equal(a, b.cpu())
        one, _ = ops.sample_tokens(x[123:124].cuda(), u[123:124].cuda(), s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0))
        assert int(one) == int(a[123])


def test_frequencies_follow_the_distribution():
    """Even random numbers draw every token as often as its probability says, to one draw."""
    x, _ = logits_of(1, 300, 16, torch.float32, spread=1.0)
    n = 20000
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    tok, lp = ops.sample_tokens(x.cuda().expand(n, -1), u.cuda(), 1.3, 100, 0.9)
    got = torch.bincount(tok.cpu(), minlength=300).double() / n
    for token in range(300):
        on = tok.cpu() == token
        if on.any():
            assert abs(float(got[token]) - math.exp(float(lp.cpu()[on][0]))) <= 1.0001 / n + 1e-6
    assert abs(float(got.sum()) - 1) < 1e-12 and (got > 0).sum() < 100


def test_streams_and_graphs():
    x, u = logits_of(8, 30011, 17)
    xd, ud = x.cuda(), u.cuda()
    want = check(x, u, k=50, p=0.9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tok, _ = ops.sample_tokens(xd, ud, 1.0, 50, 0.9)
    s.synchronize()
    assert torch.equal(tok.cpu(), want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, lp = ops.sample_tokens(xd, ud, 1.0, 50, 0.9)
    for seed in (18, 19):
        x2, u2 = logits_of(8, 30011, seed)
        xd.copy_(x2)
        ud.copy_(u2)
        g.replay()
        torch.cuda.synchronize()
        got = tok.cpu().clone()
        assert torch.equal(got, check(x2, u2, k=50, p=0.9))


def test_nothing_to_draw():
    tok, lp = ops.sample_tokens(torch.empty(0, 10, device="cuda"), torch.empty(0, device="cuda"))
    assert tok.shape == lp.shape == (0,) and tok.dtype == torch.int64 and lp.dtype == torch.float32


def test_refusals():
    x, u = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")
    bad = [(x.half(), u), (x[0], u), (x.t(), u[:1]), (x, u[:3]), (x, u.half()), (x, u.cpu()), (x[:, :0], u),
           (x.cpu(), u)]
    for a, b in bad:
        with pytest.raises((ValueError, RuntimeError)):
            ops.sample_tokens(a, b)
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=1.5),
               dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan), dict(top_k=-1),
               dict(temperature=torch.ones(3, device="cuda")), dict(top_k=torch.ones(4, device="cuda")),
               dict(top_p=torch.ones(4, dtype=torch.float64, device="cuda")), dict(min_p=torch.ones(4))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.sample_tokens(x, u, **kw)
    with pytest.raises(RuntimeError):
        ops.sample_tokens(torch.zeros(1, 2 ** 18 + 1, device="cuda"), u[:1])
