"""Sampling at the ends of what its settings may be (bars: see ``test_gpu_sample.py``)."""

import math

import pytest
import torch

from nki_moe_b200 import ops
from tests.test_gpu_sample import drawn, logits_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def spiked(rows, vocab, top, rest):
    x = torch.full((rows, vocab), rest)
    x[torch.arange(rows), torch.arange(rows) * 7 % vocab] = top
    return x


# a largest logit and many that weigh 2^-60 to 2^-64 of it: together they are what lies between top_p and 1
SPIKES = [(0.0, -42.0, 1001), (0.0, -42.0, 2040), (0.0, -42.0, 5001), (0.0, -43.5, 30001), (42.0, 1e-10, 5001),
          (-1.0, -43.25, 1001), (1.5, -41.0, 301)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p", [1 - 2.0 ** -53, 1 - 1e-15, 1 - 1e-14])
@pytest.mark.parametrize("rows", [3, 160])
def test_top_p_just_below_one_with_one_large_logit(rows, p, dtype):
    u = torch.linspace(0.0, 0.999, rows, dtype=torch.float64)
    for top, rest, vocab in SPIKES:
        x = spiked(rows, vocab, top, rest).to(dtype)
        ops.sample_tokens(x.cuda(), u.cuda(), 1.0, 1 + vocab // 2)  # another border before
        left = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
        del left  # (where the tokens may come to lie)
        tok, lp = ops.sample_tokens(x.cuda(), u.cuda(), 1.0, 0, p)
        # what is cut, and all that is left of the small ones, is 2^-42 of the sum at most
        assert torch.equal(tok.cpu(), torch.arange(rows) * 7 % vocab), (top, rest, vocab)
        assert float(lp.abs().max()) <= 2.0 ** -42 + vocab * 2.0 ** -45
        last, _ = ops.sample_tokens(x.cuda(), torch.full((rows,), math.nextafter(1.0, 0.0), dtype=torch.float64).cuda(),
                                    1.0, 0, p)
        assert int(last.min()) >= 0 and int(last.max()) < vocab


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [0.2, 0.3, 0.25])
def test_top_p_just_below_one(t, dtype):
    """Of ordinary rows; what is cut is 1e-14 of the sum at most, so tokens are those of the whole row."""
    x, u = logits_of(6, 151936, 31, dtype)
    want = [drawn(x[i], u[i].item(), t) for i in range(6)]
    assert min(w[2] for w in want) > 2 ** -31
    for p in (1 - 2.0 ** -53, 1 - 1e-15, 1 - 3e-15, 1 - 1e-14):
        left = torch.full((6,), -7, dtype=torch.int64, device="cuda")
        del left
        tok, lp = ops.sample_tokens(x.cuda(), u.cuda(), t, 0, p)
        assert tok.tolist() == [w[0] for w in want], p
        for a, (_, b, _) in zip(lp.tolist(), want):
            assert abs(a - b) <= 2 ** -24 * abs(b) + 151936 * 2 ** -45 + 1e-12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("s", [dict(), dict(min_p=1e-4), dict(top_k=3000), dict(top_p=0.97), dict(top_k=900, min_p=0.002)])
def test_a_token_for_every_random_number(s, dtype):
    """The sums of groups, of a group's vectors and of a vector's logits, each formed where it is
    needed, have to be the same whole numbers: else a number between them finds no token."""
    n = 4096
    g = torch.Generator().manual_seed(41)
    x, _ = logits_of(1, 20011, 40, dtype)
    u = torch.cat([(torch.arange(n, dtype=torch.float64) + 0.5) / n, torch.rand(n, generator=g, dtype=torch.float64)])
    u = u.sort().values.cuda()
    for rows in (2, 100, 2 * n):  # slices, parts of rows in global memory, whole rows
        for at in range(0, 2 * n, rows) if rows > 2 else (0, 17, 5000):
            part = u[at:at + rows]
            tok, lp = ops.sample_tokens(x.cuda().expand(len(part), -1), part, 0.9, **s)
            assert int(tok.min()) >= 0 and int(tok.max()) < 20011 and not lp.isnan().any()
            assert (tok.diff() >= 0).all()  # as the random numbers rise, so do the ids
            assert (x[0].cuda()[tok] > -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 200])
def test_weights_that_round_to_the_largest_are_at_least_as_large(rows, dtype):
    """Near zero logits may differ by less than their weights can."""
    g = torch.Generator().manual_seed(51)
    x = -torch.rand(rows, 2011, generator=g) * 10.0 ** -torch.randint(17, 30, (rows, 2011), generator=g)
    x[:, 1000:] -= 1.0
    x[:, 7] = 0.0
    x = x.to(dtype)
    u = torch.rand(rows, generator=g, dtype=torch.float64)
    for t in (1.0, 3.0, math.inf):
        temperature = torch.full((rows,), t, device="cuda")
        tok, lp = ops.sample_tokens(x.cuda(), u.cuda(), temperature, 0, 1.0, 1.0)
        for i in range(0, rows, 11):
            want, want_lp, _ = drawn(x[i], u[i].item(), t, 0, 1.0, 1.0)
            assert int(tok[i]) == want
            assert abs(float(lp[i]) - want_lp) <= 2 ** -24 * abs(want_lp) + 2011 * 2 ** -45 + 1e-12
