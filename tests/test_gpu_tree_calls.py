"""GPU: calls of the tree operators as a serving loop makes them: captured and replayed, in and out of inference
mode, over padded batches, strided tables, caches beyond 32-bit offsets, nothing at all and very many trees.
"""
import random

import pytest
import torch
from test_gpu_decode import BF16, E4M3, Cache, check, quantise
from test_gpu_draft_trees import _gen, _i32, above, attend, keep_plain, masks_of, tables, tree, tree_attention_64, \
    walk_64, words_of

pytestmark = pytest.mark.gpu


def _model(**kw):
    from test_gpu_lm_extend import _model

    return _model(**kw)


def _filled(cfg, model, dtype=BF16, prompt=18, seed=0):
    cache = model.new_cache(24, page_size=16, dtype=dtype)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(seed))[:15].view(3, 5).int().cuda()
    ids = torch.randint(0, cfg.vocab, (3 * prompt,), device="cuda", generator=_gen(seed))
    model.extend(ids, cache, table, _i32([prompt] * 3))
    return cache, table, _i32([prompt] * 3)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("N", [6, 30])
def test_a_captured_step_with_trees(dtype, N):
    """Replayed with other tokens, trees and lengths, it does what an eager step does."""
    cfg, model = _model(layers=3)
    rng = random.Random(N)
    steps = [dict(last=torch.randint(0, cfg.vocab, (3,), device="cuda", generator=_gen(i)),
                  drafts=torch.randint(0, cfg.vocab, (3, N), device="cuda", generator=_gen(9 + i)).int(),
                  parents=_i32([[rng.randrange(j) for j in range(1, N + 1)] for _ in range(3)]),
                  u=torch.rand((3, 4), device="cuda", generator=_gen(5 + i))) for i in range(3)]
    cache, table, lengths = _filled(cfg, model, dtype)
    eager_cache, _, eager_lengths = _filled(cfg, model, dtype)
    held = {k: v.clone() for k, v in steps[0].items()}
    run = lambda s, c, n: model.verify_tree(s["last"], s["drafts"], s["parents"], s["u"], c, table, n)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held, cache, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held, cache, lengths)
    restored, _, first = _filled(cfg, model, dtype)
    for x, y in ((cache.k, restored.k), (cache.v, restored.v), (cache.k_scale, restored.k_scale),
                 (cache.v_scale, restored.v_scale)):
        if x is not None:
            x.copy_(y)
    lengths.copy_(first)
    for s in steps:
        for k in held:
            held[k].copy_(s[k])
        graph.replay()
        want = run(s, eager_cache, eager_lengths)
        for x, y in zip(out, want):
            assert torch.equal(x, y)
        lengths.copy_(out[2])
        eager_lengths = want[2]
        for b in range(3):
            for t in range(int(want[2][b])):
                at = (table[b, t // 16].long(), t % 16)
                assert torch.equal(cache.k[:, at[0], :, at[1]].view(torch.uint8),
                                   eager_cache.k[:, at[0], :, at[1]].view(torch.uint8))
    cache.check()


@pytest.mark.parametrize("first,then", [(True, False), (False, True)])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_trees_in_and_out_of_inference_mode(first, then, dtype):
    cfg, model = _model()
    with torch.inference_mode(first):
        cache, table, lengths = _filled(cfg, model, dtype)
    drafts, parents = _i32([[3, 4, 5, 6]] * 3), _i32([0, 0, 1, 2])
    u = torch.full((3, 3), 0.5, device="cuda")
    out = []
    for mode in (first, then, first):
        with torch.inference_mode(mode):
            out.append([x.clone() for x in model.verify_tree(_i32([1, 2, 3]), drafts, parents, u, cache, table, lengths)])
            cache.check()
    for x in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], x))


@pytest.mark.parametrize("max_q", [5, None])
def test_rows_behind_the_last_tree(max_q):
    """A padded batch gives its trees' rows the logits that they have without the padding."""
    cfg, model = _model()
    parents = [-1, 0, 0, 1, 2] + [-1, 0, 1] + [-1]
    start = [0, 5, 8, 9]
    ids = torch.randint(0, cfg.vocab, (9,), device="cuda", generator=_gen(3))
    got = []
    for pad in (0, 23):
        cache, table, lengths = _filled(cfg, model)
        padding = torch.zeros(pad, dtype=torch.long, device="cuda")
        logits = model.extend(torch.cat([ids, padding]), cache, table, lengths + _i32([5, 3, 1]), _i32(start), max_q,
                              parents=_i32(parents + [7] * pad))
        assert bool(torch.isfinite(logits).all())
        got.append((logits[:9], cache))
        cache.check()
    # other row counts go through other tilings of the projections: the sizes of bf16 activations' steps
    diff = (got[0][0].float() - got[1][0].float()).abs().max()
    assert float(diff) <= 0.05 * float(got[0][0].float().abs().max())
    b = 0
    for t in range(23):  # layer 0's keys do not hang on them
        at = (table[b, t // 16].long(), t % 16)
        assert float((got[0][1].k[0, at[0], :, at[1]].float() - got[1][1].k[0, at[0], :, at[1]].float()).abs().max()) \
            <= 0.05 * float(got[0][1].k[0, at[0]].float().abs().max())


def test_nothing_to_do():
    import computd_b200 as cb

    k = torch.zeros((4, 2, 16, 64), dtype=BF16, device="cuda")
    none = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    cos, sin = tables(4, 64, torch.float32)
    slots = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert cb.kv_cache_append(none, none, none, cos, sin, k, k.clone(), slots).shape == (0, 2, 64)
    assert cb.kv_cache_append(None, none, none, cos[:0], sin[:0], k, k.clone(), slots) is None
    table = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    cb.kv_cache_keep(k, k.clone(), table, _i32([]), torch.zeros((0, 2), dtype=torch.int32, device="cuda"), _i32([]))
    mask = torch.zeros((0, 1), dtype=torch.int64, device="cuda")
    for b in (0, 2):
        table, lengths = torch.zeros((b, 3), dtype=torch.int32, device="cuda"), _i32([7] * b)
        assert cb.paged_tree_attention(none, k, k, table, lengths, mask, q_start=_i32([0] * (b + 1))).shape == (0, 2, 64)
    assert cb.tree_masks(_i32([]), q_start=_i32([0, 0]))[0].shape == (0, 1)
    assert not bool(k.any())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [9, 30, 50, 90])
def test_tables_that_lie_apart(kind, n):
    """A row of pages is part of a longer one."""
    import computd_b200 as cb

    cache = Cache(kind, [150, 333], 2, 64, 16, seed=n)
    q, seen = torch.randn((2 * n, 2, 64), device="cuda", generator=_gen(n)).to(BF16), masks_of([n, n], "tree", 1)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    wide = torch.full((2, 3, cache.table.shape[1]), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, 1] = cache.table
    got = cb.paged_tree_attention(q, cache.k, cache.v, wide[:, 1], cache.len, words_of(seen, -(-n // 64)),
                                  **cache.scales())
    check(got, want, mag)
    path = [[0, 3, 7], [0, 1, 5]]
    expect = [x.clone()[None] for x in (cache.k, cache.v, *cache.scales().values())]
    keep_plain(expect, cache.table.tolist(), [100, 200], path, [2, 1], 16)
    cb.kv_cache_keep(cache.k, cache.v, wide[:, 1], _i32([100, 200]), _i32(path), _i32([2, 1]), **cache.scales())
    for x, y in zip((cache.k, cache.v, *cache.scales().values()), expect):
        assert torch.equal(x.view(torch.uint8), y[0].view(torch.uint8))


def test_very_many_trees():
    """More than 65535 of them: of one to three nodes."""
    import computd_b200 as cb

    rng = random.Random(0)
    B, V = 70000, 5
    sizes = [rng.randint(0, 3) for _ in range(B)]
    start = [0]
    for n in sizes:
        start.append(start[-1] + n)
    trees = [tree(n, rng) for n in sizes]
    flat = [p for t in trees for p in t]
    mask, depth = cb.tree_masks(_i32(flat), q_start=_i32(start), max_q=3)
    seen = [s for t in trees for s in above(t)]
    assert torch.equal(mask, torch.tensor([[sum(1 << j for j in s)] for s in seen], device="cuda"))
    assert torch.equal(depth, _i32([len(s) - 1 for s in seen]))
    p = torch.rand((len(flat), V), device="cuda", generator=_gen(1))
    tokens = torch.randint(0, V, (len(flat),), device="cuda", generator=_gen(2)).int()
    u = torch.rand((B, 3), device="cuda", generator=_gen(3))
    kept, out, path = cb.verify_tree(p, tokens, _i32(flat), u, q_start=_i32(start))
    some = rng.sample(range(B), 200) + [0, B - 1]
    for b in some:
        want = walk_64(p[start[b]:start[b + 1]], tokens[start[b]:start[b + 1]].tolist(), trees[b], u[b:b + 1].cpu(),
                       [0, sizes[b]])
        assert (kept[b:b + 1].tolist(), out[b:b + 1].tolist(), path[b:b + 1].tolist()) == tuple(want)
    # and their paths kept, on a page each
    k = torch.randn((B, 1, 16, 16), device="cuda", generator=_gen(4)).to(BF16)
    v, old = k.clone(), k.clone()
    table = torch.arange(B, device="cuda", dtype=torch.int32)[:, None]
    cb.kv_cache_keep(k, v, table, _i32([5] * B), path, torch.where(path[:, 0] < 0, -1, kept))
    at = torch.arange(3, device="cuda")
    move = (at <= kept[:, None]) & (path >= 0)
    want = old.clone()
    b, i = move.nonzero(as_tuple=True)
    want[b, :, 5 + i] = old[b, :, 5 + path[b, i].long()]
    assert torch.equal(k, want) and torch.equal(v, want)


def test_cache_beyond_32_bit_offsets():
    """A cache of 5 GB for keys and as much for values: trees are appended to its last pages, attended to, and their
    paths kept there."""
    import computd_b200 as cb

    heads, page, d = 8, 64, 128
    n_pages = 5 * 2 ** 30 // (heads * page * d)
    kc, vc = (torch.zeros((n_pages, heads, page, d), device="cuda", dtype=E4M3) for _ in range(2))
    ks, vs = (torch.zeros((n_pages, heads, page), device="cuda") for _ in range(2))
    T = 200
    k, v = (torch.randn((T, heads, d), device="cuda", generator=_gen(i)).to(BF16) for i in range(2))
    pages = _i32([n_pages - 1, n_pages // 2 + 5, 3, n_pages - 2])
    t = torch.arange(T, device="cuda")
    slots = pages.long()[t // page] * page + t % page
    cos, sin = torch.ones((T, d // 2), device="cuda"), torch.zeros((T, d // 2), device="cuda")
    cb.kv_cache_append(None, k, v, cos, sin, kc, vc, slots, k_scale=ks, v_scale=vs)
    apart = torch.cat([k[..., 0::2], k[..., 1::2]], -1)  # no rotation but the order of channels
    for got, scale, x in ((kc, ks, apart), (vc, vs, v)):
        codes, want = quantise(x)
        at = (pages.long()[t // page], slice(None), t % page)
        assert torch.equal(got[at].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale[at], want)
    cache = Cache.__new__(Cache)
    cache.k, cache.v, cache.k_scale, cache.v_scale = kc, vc, ks, vs
    cache.table, cache.page, cache.lengths = pages[None], page, [T]
    cache.len = _i32([T])
    for n in (5, 30, 60, 100):
        q = torch.randn((n, heads, d), device="cuda", generator=_gen(n)).to(BF16)
        seen = masks_of([n], "tree", n)
        check(attend(cache, q, [n], seen), *tree_attention_64(q, cache, [0, n], seen))
    path = [0, 40, 41, 70]
    before = [x[pages[(100 + p) // page].long(), :, (100 + p) % page].clone() for x in (kc, vc, ks, vs) for p in path]
    cb.kv_cache_keep(kc, vc, pages[None], _i32([100]), _i32([path]), _i32([3]), k_scale=ks, v_scale=vs)
    after = [x[pages[(100 + i) // page].long(), :, (100 + i) % page] for x in (kc, vc, ks, vs) for i in range(4)]
    assert all(torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(before, after))
