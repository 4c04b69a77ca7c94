"""Lengths that make no sense in the calls of drafted decoding: they are reported, nothing outside
of what was given is read or written, and what is documented for the others holds."""

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


def recycled(T):
    """Leaves a block of 7s behind, of the size that the next outputs take."""
    for dtype in (torch.int32, torch.int64):
        blocks = [torch.full((T,), 7, dtype=dtype, device="cuda") for _ in range(4)]
        del blocks


@pytest.mark.parametrize("starts,lens,paths", [
    ([0, 65, 69], [70, 20], {1: [65, 66, 67, 68]}),  # more nodes than a tree has
    ([0, 4, 8], [3, 20], {1: [4, 5, 6, 7]}),  # a cache shorter than the tree
    ([0, 4, 8], [20, 10 ** 6], {0: [0, 1, 2, 3]}),
    ([5, 9, 9, 12], [20, 0, 20], {0: [5, 6, 7, 8], 2: [9, 10, 11]}),  # rows before the first
    ([-3, 4, 8], [20, 20], {1: [4, 5, 6, 7]}),
    ([3, 7, 10 ** 9], [20, 20], {0: [3, 4, 5, 6]}),
    ([6, 2], [20], {}),
    ([-8, -4], [20], {}),
    ([100, 104], [20], {}),
])
def test_rows_without_a_path_are_minus_one(starts, lens, paths, monkeypatch):
    """Of refused sequences, and of none."""
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    T, B = 80, len(lens)
    token = torch.ones(T, dtype=torch.int64, device="cuda")
    parents = torch.full((T,), -1, dtype=torch.int32)
    for rows in paths.values():
        parents[rows] = torch.arange(-1, len(rows) - 1, dtype=torch.int32)  # chains that are agreed with
    pages = torch.zeros(2, 5 * B, 1, 16, 8, dtype=torch.bfloat16, device="cuda")
    table = torch.arange(5 * B, dtype=torch.int32, device="cuda").view(B, 5)
    want = torch.full((T,), -1, dtype=torch.int32)
    for rows in paths.values():
        want[rows] = torch.arange(len(rows), dtype=torch.int32)
    recycled(T)
    counts, path, new = ops.accept_drafts(token, token, parents.cuda(), ints(*starts), ints(*lens), pages, table)
    refused = [b for b in range(B) if b not in paths and starts[b] != starts[b + 1]]
    if refused:
        reported()
    assert counts.tolist() == [len(paths.get(b, [])) for b in range(B)]
    assert torch.equal(path.cpu(), want)
    assert torch.equal(new.cpu(), torch.where(want >= 0, 1, -1))


@pytest.mark.parametrize("starts,paths", [
    ([0, 70, 4, 8], {2: [4, 5, 6, 7]}),  # the first would have what the third has
    ([0, 4, 8, 2], {0: [0, 1, 2, 3], 1: [4, 5, 6, 7]}),  # and what lies behind the last
    ([6, 2, 9, 9], {1: [2, 3, 4, 5, 6, 7, 8]}),  # and before the first
])
def test_rows_of_others_are_left_to_them(starts, paths, monkeypatch):
    """Where starts do not rise, a refused sequence's rows may be another's."""
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    for _ in range(5):
        test_rows_without_a_path_are_minus_one(starts, [70] * 3, paths, monkeypatch)


def test_calls_of_no_sequences_and_of_no_rows():
    """Through the C entry: the outputs are written all the same."""
    from nki_moe_b200 import _lib

    tok = torch.ones(9, dtype=torch.int64, device="cuda")
    pages = torch.zeros(1, 2, 1, 16, 8, dtype=torch.bfloat16, device="cuda")
    table, status = ints(0, 1).view(1, 2), torch.zeros(64, dtype=torch.int32, device="cuda")
    for T, B in ((9, 0), (0, 1)):
        counts, path, new = ints(7), ints(*[7] * 9), torch.full((9,), 7, dtype=torch.int64, device="cuda")
        _lib.call("nkimoe_accept_drafts", tok.data_ptr(), tok.data_ptr(), path.data_ptr(), ints(0, 0).data_ptr(),
                  ints(0).data_ptr(), pages.data_ptr(), 1, 2, 1, 16, 16, table.data_ptr(), 2, 2, counts.data_ptr(),
                  path.data_ptr(), new.data_ptr(), T, B, status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert (path.tolist(), new.tolist()) == (([-1] * 9,) * 2 if B == 0 else ([7] * 9,) * 2)
        assert counts.tolist() == [7 if B == 0 else 0]
