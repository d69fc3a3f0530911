"""GPU: kv_cache_keep of paths longer than a look at three nodes, of one layer by itself, and in
caches whose pages and layers lie apart."""
import random

import pytest
import torch
from test_gpu_decode import BF16, E4M3, quantise
from test_gpu_draft_trees import _gen, _i32, keep_plain

pytestmark = pytest.mark.gpu


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == E4M3 else x


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


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers", [None, 1, 3])
@pytest.mark.parametrize("H,d,page,n,steps", [(2, 80, 16, 40, 7), (1, 16, 128, 600, 300), (3, 128, 32, 64, 12)])
def test_layers_and_pages_that_lie_apart(kind, layers, H, d, page, n, steps):
    """`layers` None: one layer's caches, of four dimensions.  Nothing between the pages changes."""
    import computd_b200 as cb

    rng = random.Random(n)
    B, each = 4, -(-(n + 20) // page) + 1
    L, pages = layers or 1, B * each + 1
    wide = []
    for seed in (1, 2):
        x = torch.randn((L, 2, pages, 3, H, page, d), device="cuda", generator=_gen(seed)).to(BF16)
        wide.append(x)
    if kind == "e4m3":
        (k, ks), (v, vs) = quantise(wide[0]), quantise(wide[1])
        wide = [k, v, ks, vs]
    before = [x.clone() for x in wide]
    views = [x[:, 1, :, 2] for x in wide]  # every other layer, every third page
    assert not any(x.is_contiguous() for x in views)
    table = torch.randperm(pages, device="cuda", generator=_gen(3))[:B * each].view(B, each).int()
    start = [rng.randrange(20) for _ in range(B)]
    kept = [min(steps, n) - 1, -1, rng.randrange(1, steps), rng.randrange(1, steps)]
    path = [sorted(rng.sample(range(n), max(m, 0) + 1)) for m in kept]
    want = [x.clone() for x in views]
    keep_plain(want, table.tolist(), start, path, kept, page)
    assert not torch.equal(_bytes(want[0]), _bytes(views[0]))
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    args = views if layers else [x[0] for x in views]
    scales = dict(zip(("k_scale", "v_scale"), args[2:]))
    cb.kv_cache_keep(args[0], args[1], table, _i32(start), _i32([p + [-1] * (steps - len(p)) for p in path]),
                     _i32(kept), status=status, **scales)
    assert int(status) == 0
    for x, y, w, old in zip(views, want, wide, before):
        assert torch.equal(_bytes(x), _bytes(y))
        x.copy_(old[:, 1, :, 2])
        assert torch.equal(_bytes(w), _bytes(old))
