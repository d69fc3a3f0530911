"""GPU: attention of many trees at once, where its blocks have whole sequences, and of few over long contexts,
where blocks share the keys of one; against the plain formulas in 64 bits.

The tolerance is test_gpu_decode.py's, which holds here too: over e4m3 caches queries are rounded to 2^-18 of their
row's largest value, which moves a score by less than 2^-12, and weights times their values' scales to
2^-12, or where those lie below 2^-24 of the largest by what is below 2^-25 each of codes up to 448.
"""
import math
import random

import pytest
import torch
from test_gpu_decode import BF16, Cache, check, starts
from test_gpu_draft_trees import _gen, _i32, attend, masks_of, tree_attention_64, words_of

pytestmark = pytest.mark.gpu


def many(kind, rows, group, d, page, longest, seed, kv_heads=16, batch=24):
    """Trees of up to `rows` rows per key/value head, over up to `longest` tokens."""
    rng = random.Random(seed)
    most = rows // group
    new = [most] + [rng.randint(1, most) for _ in range(batch - 1)]
    lengths = [longest] + [rng.randint(n, longest) for n in new[1:]]
    new[3], lengths[5], new[7], lengths[7] = 0, 0, most, max(most // 2, 1)  # no tree; no token; more nodes than tokens
    cache = Cache(kind, lengths, kv_heads, d, page, seed=seed)
    q = torch.randn((sum(new), kv_heads * group, d), device="cuda", generator=_gen(seed)).to(BF16)
    return cache, q, new


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [17, 32, 33, 48, 64])
@pytest.mark.parametrize("group,d,page,longest", [(1, 128, 64, 1000), (1, 80, 32, 700), (4, 64, 16, 129), (2, 128, 128, 128),
                                                  (1, 16, 16, 1024), (8, 112, 64, 385), (1, 64, 128, 60)])
@pytest.mark.parametrize("masks", ["tree", "any"])
def test_many_trees(kind, rows, group, d, page, longest, masks):
    cache, q, new = many(kind, rows, group, d, page, max(longest, rows // group), seed=rows + d)
    seen = masks_of(new, masks, rows)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = attend(cache, q, new, seen, status=status)
    check(got, *tree_attention_64(q, cache, starts(new), seen))
    assert int(status) == 0
    assert torch.equal(got, attend(cache, q, new, seen))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [20, 64])
def test_more_trees_than_are_ranked(kind, rows):
    cache, q, new = many(kind, rows, 1, 64, 16, 260, seed=9, kv_heads=2, batch=150)
    seen = masks_of(new, "tree", 1)
    check(attend(cache, q, new, seen), *tree_attention_64(q, cache, starts(new), seen))


@pytest.mark.parametrize("d,heads,kv_heads,most", [(112, 64, 16, 100), (80, 192, 24, 33), (128, 16, 16, 200), (64, 64, 16, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences_without_cached_tokens_get_zeros(d, heads, kv_heads, most, causal):
    """Among many others, of more rows than one block takes at once."""
    import computd_b200 as cb

    rng = random.Random(d)
    new = [rng.randint(most // 2, most) for _ in range(140)]
    lengths = [0 if rng.random() < 0.5 else rng.randint(1, 130) for _ in new]
    cache = Cache("bf16", lengths, kv_heads, d, 64, seed=d)
    q = torch.randn((sum(new), heads, d), device="cuda", generator=_gen(d)).to(BF16)
    start, mask = _i32(starts(new)), None if causal else words_of(masks_of(new, "tree", 3), -(-most // 64))
    empty = torch.repeat_interleave(cache.len == 0, torch.tensor(new, device="cuda"))
    for _ in range(5):
        if causal:
            got = cb.paged_attention(q, cache.k, cache.v, cache.table, cache.len, q_start=start, max_q=most)
        else:
            got = cb.paged_tree_attention(q, cache.k, cache.v, cache.table, cache.len, mask, q_start=start, max_q=most)
        assert bool((got[empty] == 0).all()) and not bool(torch.isnan(got).any())


@pytest.mark.parametrize("rows", [24, 60, 128, 300])
@pytest.mark.parametrize("lengths", [[700] * 3, [5000, 130, 2100], [20000], [1300, 9000, 1, 400]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_few_trees_share_their_keys(kind, rows, lengths):
    """Contexts cut into parts, ragged ones and a sequence alone."""
    new = [min(rows // 2, n) for n in lengths]
    cache = Cache(kind, lengths, 3, 128, 64, seed=rows)
    q = torch.randn((sum(new), 6, 128), device="cuda", generator=_gen(rows)).to(BF16)
    seen = masks_of(new, "tree", 2)
    check(attend(cache, q, new, seen), *tree_attention_64(q, cache, starts(new), seen))


@pytest.mark.parametrize("heads,length", [(48, 700), (3, 3000)])
@pytest.mark.parametrize("rows", [12, 30, 60, 100])
def test_scales_far_apart(heads, length, rows):
    """Values' scales over 24 powers of two, keys' over four."""
    cache = Cache("e4m3", [length, length // 2], heads, 128, 64, seed=5, poison=False)
    g = _gen(11)
    cache.v_scale *= 2.0 ** torch.randint(-12, 13, cache.v_scale.shape, device="cuda", generator=g)
    cache.k_scale *= 2.0 ** torch.randint(-2, 2, cache.k_scale.shape, device="cuda", generator=g)
    q = torch.randn((2 * rows, heads, 128), device="cuda", generator=g).to(BF16)
    seen = masks_of([rows, rows], "tree", 4)
    check(attend(cache, q, [rows, rows], seen), *tree_attention_64(q, cache, [0, rows, 2 * rows], seen))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,length", [(17, 17), (24, 500), (33, 700), (64, 129)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_a_node_may_not_see_does_not_reach_it(kind, d, n, length, bad):
    heads = 64
    cache = Cache(kind, [length], heads, d, 16, seed=n, poison=False)
    q = torch.randn((n, heads, d), device="cuda", generator=_gen(6)).to(BF16)
    rng = random.Random(n)
    seen = masks_of([n], "any", 9)
    hidden = {rng.randrange(n) for _ in range(1 + n // 6)}
    for s in seen[:n // 2]:
        s -= hidden
    clean, mag = tree_attention_64(q, cache, [0, n], seen)
    for j in hidden:
        page, off = int(cache.table[0, (length - n + j) // 16]), (length - n + j) % 16
        if kind == "e4m3":
            cache.k_scale[page, :, off] = bad
            cache.v_scale[page, :, off] = bad
        else:
            cache.k[page, :, off] = bad
            cache.v[page, :, off, [1, d - 2]] = bad
    got = attend(cache, q, [n], seen)
    blind = torch.tensor([not (s & hidden) for s in seen], device="cuda")
    check(got[blind], clean[blind], mag[blind])
    assert not bool(torch.isfinite(got[~blind]).all(-1).any())


@pytest.mark.parametrize("n,length", [(24, 500), (64, 700)])
def test_values_that_are_not_finite_reach_who_sees_them(n, length):
    heads, d = 64, 80
    cache = Cache("bf16", [length], heads, d, 16, seed=n, poison=False)
    q = torch.randn((n, heads, d), device="cuda", generator=_gen(6)).to(BF16)
    seen = masks_of([n], "any", 10)
    clean, mag = tree_attention_64(q, cache, [0, n], seen)
    bad = {n // 3: 3, n - 1: d - 1}  # node: channel
    for j, c in bad.items():
        at = length - n + j
        cache.v[int(cache.table[0, at // 16]), :, at % 16, c] = math.nan
    got = attend(cache, q, [n], seen)
    expect = torch.zeros((n, heads, d), dtype=torch.bool, device="cuda")
    for r, s in enumerate(seen):
        for j, c in bad.items():
            if j in s:
                expect[r, :, c] = True
    assert torch.equal(torch.isnan(got), expect)
    check(torch.where(expect, 0, got), torch.where(expect, 0, clean), mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [20, 50])
@pytest.mark.parametrize("heads", [2, 64])
def test_pages_lengths_and_sizes_are_reported(kind, n, heads):
    import computd_b200 as cb

    cache = Cache(kind, [200, 200], heads, 64, 16, seed=3)
    q = torch.randn((2 * n, heads, 64), device="cuda", generator=_gen(8)).to(BF16)
    seen = masks_of([n, n], "tree")
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    for spoil in ("page", "length", "size"):
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        table, length = cache.table.clone(), cache.len.clone()
        max_q, begin = n, [0, n, 2 * n]
        if spoil == "page":
            cache.table[1, 3] = 2 ** 30
        elif spoil == "length":
            cache.len[1] = cache.table.shape[1] * 16 + 1
        else:
            max_q, begin = 18, [0, 18, 2 * n]  # more nodes in the second
        got = cb.paged_tree_attention(q, cache.k, cache.v, cache.table, cache.len, words_of(seen, 3),
                                      q_start=_i32(begin), max_q=max_q, status=status, **cache.scales())
        cache.table, cache.len = table, length
        assert int(status) == 5, spoil
        assert bool(torch.isnan(got[begin[1]:begin[2]]).all()), spoil
        if spoil != "size":
            check(got[:n], want[:n], mag[:n])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,heads,lengths", [(32, 16, [500] * 9), (30, 2, [3000, 900]), (60, 2, [3000, 900])])
def test_two_captured_calls_and_an_eager_one(kind, rows, heads, lengths):
    """Two graphs replayed on two streams, and a call between them, each with what it computed alone."""
    import computd_b200 as cb

    new = [rows] * len(lengths)
    calls = []
    for seed in (1, 2):
        cache = Cache(kind, lengths, heads, 128, 64, seed=seed)
        q = torch.randn((sum(new), heads, 128), device="cuda", generator=_gen(seed)).to(BF16)
        mask, start = words_of(masks_of(new, "tree", seed), 1), _i32(starts(new))
        calls.append(lambda c=cache, q=q, m=mask, s=start: cb.paged_tree_attention(
            q, c.k, c.v, c.table, c.len, m, q_start=s, max_q=rows, **c.scales()))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in calls]
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        between = calls[0]()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(between, want[0])
