"""GPU: tree_masks over ranges of rows that are none, descending or outside: every row of no sequence is
zeros, whatever the memory held, and the other sequences' rows are theirs."""
import random

import pytest
import torch
from test_gpu_draft_trees import _i32, above, tree, words_of

pytestmark = pytest.mark.gpu


def _want(parents, start, max_q):
    T = len(parents)
    seen = [set()] * T
    for lo, hi in zip(start, start[1:]):
        if 0 <= lo <= hi <= T and hi - lo <= max_q:
            seen[lo:hi] = above(parents[lo:hi])
    return seen


def _masks(parents, start, max_q, status):
    """The call's mask and depth, in memory that held ones before."""
    import computd_b200 as cb

    T = len(parents)
    args = _i32(parents), _i32(start)
    held = [torch.full((T, -(-max_q // 64)), -1, dtype=torch.int64, device="cuda"),
            torch.full((T,), -1, dtype=torch.int32, device="cuda")]
    torch.cuda.synchronize()
    del held  # what the outputs are most likely made of
    return cb.tree_masks(args[0], q_start=args[1], max_q=max_q, status=status)


@pytest.mark.parametrize("max_q", [40, 128, 200])
@pytest.mark.parametrize("start", [
    [0, 2, 1],                     # descends: row 2 behind the last
    [0, 9, 4, 6],                  # behind T, then descends
    [3, 2], [-1, 3], [9, 9], [5, 5, 5], [-4, -2, 0, 7],
    [5, 7, 0, 3],                  # rows before the first sequence's are the last one's
    [0, 3, 8, 3, 5],
    [2, 4, 4, 6],                  # nothing bad: rows before and behind
])
def test_rows_of_no_sequence_are_zeros(start, max_q):
    T = 7
    parents = []
    for t in range(T):  # below t whatever the range, or none
        lo = max([s for s, e in zip(start, start[1:]) if 0 <= s <= t < e <= T], default=t)
        parents.append(t - lo - 1)
    bad = any(not 0 <= lo <= hi <= T for lo, hi in zip(start, start[1:]))
    for _ in range(5):
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        mask, depth = _masks(parents, start, max_q, status)
        seen = _want(parents, start, max_q)
        assert torch.equal(mask, words_of(seen, -(-max_q // 64)))
        assert depth.tolist() == [max(len(s) - 1, 0) for s in seen]
        assert int(status) == (5 if bad else 0)


@pytest.mark.parametrize("most", [30, 150])
@pytest.mark.parametrize("B", [3, 700])
def test_many_rows_with_some_bad_ranges(most, B):
    """Gaps between, before and behind, by ranges that descend (so that the next begins earlier) or end
    outside; more rows than are told apart at a time."""
    rng = random.Random(B + most)
    T = 40 * B + 9000
    start, parents, at = [], [-1] * T, rng.randrange(1, 200)
    # a list of offsets in which every other range goes back to before the one behind it
    spans = []
    for _ in range(B // 2):
        n = rng.randint(0, most)
        if at + n > T:
            break
        spans.append((at, at + n))
        parents[at:at + n] = tree(n, rng)
        at += n + rng.choice([0, 0, 1, 50])
    rng.shuffle(spans)
    for lo, hi in spans:
        start += [lo, hi]  # hi to the next lo: descending, or a range over others' rows
    ok, taken = [], set()
    for i in range(len(start) - 1):  # ranges between the spans must be bad, or rows would be two sequences'
        lo, hi = start[i], start[i + 1]
        if i % 2 and lo <= hi:
            ok.append(i)
    for i in reversed(ok):
        start.insert(i + 1, T + 1)  # ends outside, and the next descends from there
    seen = _want(parents, start, most)
    for lo, hi in zip(start, start[1:]):
        if 0 <= lo <= hi <= T:
            assert not taken & set(range(lo, hi))
            taken |= set(range(lo, hi))
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    mask, depth = _masks(parents, start, most, status)
    assert torch.equal(mask, words_of(seen, -(-most // 64)))
    assert depth.tolist() == [max(len(s) - 1, 0) for s in seen]
