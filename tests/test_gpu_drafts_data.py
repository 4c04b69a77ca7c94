"""Lengths that make no sense at the ends of their type's range, in the calls of drafted
decoding: they are reported, and nothing outside of what was given is read or written."""

import pytest
import torch

from nki_moe_b200 import ops
from nki_moe_b200._lib import NKIMoEError
from tests.test_gpu_accept_drafts import case
from tests.test_gpu_tree import tree_case, trees_of

pytestmark = pytest.mark.gpu

LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def reported():
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    ops.read_paged_status()  # cleared


@pytest.mark.parametrize("starts", [(HIGH, LOW), (HIGH, LOW + 3), (HIGH - 5, LOW), (LOW, HIGH), (LOW, LOW + 4), (0, LOW),
                                    (4, LOW), (HIGH - 4, HIGH)])
def test_starts_at_the_ends_of_the_type(starts, monkeypatch):
    """The difference of two of them may be a small number in 32 bits."""
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    args, out = tree_case([20], trees_of([4], 1), 8, 2, 16, seed=60)
    args[4] = ints(*starts)
    out.fill_(3.0)
    ops.paged_tree_attention(*args, out=out)
    reported()
    assert (out == 3.0).all()
    args, _ = case([4], [14], 8, 1, trees=[([1, 9, 1, 1], [1] * 4, [-1, 0, 0, 2])])
    dev = [a.cuda() for a in args]
    dev[3] = ints(*starts)
    counts, _, _ = ops.accept_drafts(*dev)
    reported()
    assert counts.tolist() == [0] and torch.equal(dev[5].cpu(), args[5])


def test_starts_at_the_ends_of_the_type_among_others(monkeypatch):
    """40 sequences, so that they are looked up 32 at a time."""
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    args, out = tree_case([20 + b for b in range(40)], trees_of([3] * 40, 2), 8, 2, 16, seed=61)
    starts = args[4].clone()
    starts[20], starts[21] = HIGH, LOW
    args[4] = starts
    out.fill_(3.0)
    ops.paged_tree_attention(*args, out=out)
    reported()
    assert (out[19 * 3:22 * 3] == 3.0).all()  # the three sequences that begin or end there


@pytest.mark.parametrize("length", [HIGH, LOW, -1, 1 << 30])
def test_lengths_at_the_ends_of_the_type(length, monkeypatch):
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    args, out = tree_case([20, 30], trees_of([4, 5], 1), 8, 2, 16, seed=62)
    good = out.clone()
    args[5][0] = length
    out.fill_(3.0)
    ops.paged_tree_attention(*args, out=out)
    reported()
    assert (out[:4] == 3.0).all() and torch.equal(out[4:], good[4:])
    args, want = case([4, 4], [14, 3], 8, 1)
    dev = [a.cuda() for a in args]
    dev[4][0] = length
    counts, _, _ = ops.accept_drafts(*dev)
    reported()
    assert counts.tolist() == [0, int(want[0][1])]
