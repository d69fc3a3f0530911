"""GPU: kv_cache_keep of bad paths of many nodes."""
import pytest
import torch
from test_gpu_decode import BF16
from test_gpu_draft_trees import _gen, _i32, keep_plain

pytestmark = pytest.mark.gpu


def _bad_path(which, n):
    """An ascending path of n + 1 nodes, spoilt in one place."""
    path = list(range(0, 2 * n + 2, 2))
    if which == "falls back":  # and ascends from there, below its places
        path[n // 2:] = range(n - n // 2 + 1)
    elif which == "below -1":  # ascends too
        path = list(range(-9, n - 8))
    elif which == "starts below":
        path[0] = -1
    elif which == "twice":
        path[n // 2] = path[n // 2 - 1]
    elif which == "small steps":  # every pair ascends but the last, whose place is behind its node
        path = list(range(n)) + [n - 1]
    return path


@pytest.mark.parametrize("which", ["falls back", "below -1", "starts below", "twice", "small steps"])
@pytest.mark.parametrize("n", [2, 40, 254, 257, 700])
@pytest.mark.parametrize("start", [0, 5])
@pytest.mark.parametrize("pages_of", ["just its own", "the last row"])
def test_bad_paths_are_reported_and_move_nothing(which, n, start, pages_of):
    """Their places may lie behind the sequence's pages, and behind the table."""
    import computd_b200 as cb

    path = _bad_path(which, n)
    pages = max(-(-(start + max(path) + 1) // 16), 1)  # no more than the path's own nodes need
    k = torch.randn((2 * pages, 1, 16, 16), device="cuda", generator=_gen(n)).to(BF16)
    v = torch.randn((2 * pages, 1, 16, 16), device="cuda", generator=_gen(n + 1)).to(BF16)
    table = torch.arange(2 * pages, device="cuda", dtype=torch.int32).view(2, pages)
    good = [0, 2] + [-1] * (len(path) - 2)
    rows, kept = ([good, path], [1, n]) if pages_of == "the last row" else ([path, good], [n, 1])
    want = [k.clone()[None], v.clone()[None]]
    keep_plain(want, table.tolist(), [start] * 2, rows, [x if p is good else -1 for x, p in zip(kept, rows)], 16)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    cb.kv_cache_keep(k, v, table, _i32([start] * 2), _i32(rows), _i32(kept), status=status)
    assert int(status) == 5 and torch.equal(k, want[0][0]) and torch.equal(v, want[1][0])
