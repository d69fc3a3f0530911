"""GPU: the operators of trees of drafted tokens (include/dwa_decode.h) against plain formulas in
64 bits: masks, append with rotation, attention, walk, keep, and a run of them together.

The attention's tolerance is test_gpu_decode.py's.  Append: an output's f32 value is off by at
most 2^-23 of itself and 2^-46 of its products (their rounding errors are carried along), and is then
rounded once: to bf16 (2^-8 of the value), or relative to the scale s to e4m3 (2^-4 of the value, and
2^-10 s where codes are subnormal, the half of their step 2^-9).
"""
import math
import random

import pytest
import torch
from test_gpu_decode import BF16, E4M3, Cache, check, quantise, starts

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tree(n, rng, deep=False):
    return [-1] + [i - 1 if deep and rng.random() < 0.8 else rng.randrange(i) for i in range(1, n)] if n else []


def above(parents):
    """The set of every node and its ancestors."""
    got = []
    for i, p in enumerate(parents):
        got.append({i} | (got[p] if p >= 0 else set()))
    return got


def words_of(seen, words):
    """Rows of bits as int64 words."""
    got = torch.zeros((len(seen), words), dtype=torch.int64)
    for r, nodes in enumerate(seen):
        for w in range(words):
            x = sum(1 << (j - 64 * w) for j in nodes if 64 * w <= j < 64 * w + 64)
            got[r, w] = x - (1 << 64) if x >> 63 else x
    return got.cuda()


# ---------------------------------------------------------------- masks
@pytest.mark.parametrize("sizes", [[1], [5, 0, 64, 65, 1], [128, 3], [200], [1000, 17]])
@pytest.mark.parametrize("deep", [False, True])
def test_tree_masks(sizes, deep):
    import computd_b200 as cb

    rng = random.Random(len(sizes))
    trees = [tree(n, rng, deep) for n in sizes]
    trees[-1][0] = -1
    flat = [p for t in trees for p in t]
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    mask, depth = cb.tree_masks(_i32(flat), q_start=_i32(starts(sizes)), max_q=max(sizes), status=status)
    seen = [s for t in trees for s in above(t)]
    assert torch.equal(mask, words_of(seen, -(-max(sizes) // 64)))
    assert depth.tolist() == [len(s) - 1 for s in seen] and int(status) == 0
    assert depth.dtype == torch.int32


def test_tree_masks_of_equal_trees_and_chains():
    import computd_b200 as cb

    chain = list(range(-1, 69))
    mask, depth = cb.tree_masks(_i32(chain * 3), n_trees=3)
    assert mask.shape == (210, 2) and depth.tolist() == list(range(70)) * 3
    assert torch.equal(mask, words_of([set(range(i + 1)) for i in range(70)] * 3, 2))
    one, _ = cb.tree_masks(_i32(chain))
    assert torch.equal(one, mask[:70])
    none, depth = cb.tree_masks(_i32([]))
    assert none.shape == (0, 1) and depth.shape == (0,)


def test_tree_masks_report_bad_parents_ranges_and_sizes():
    import computd_b200 as cb

    status = torch.zeros((), dtype=torch.int32, device="cuda")
    # of node 1 itself, one behind node 2, one below -1
    mask, depth = cb.tree_masks(_i32([-1, 1, 3, 0, -2, 4]), status=status)
    assert int(status) == 5 and mask[:, 0].tolist() == [1, 2, 4, 9, 16, 48]
    assert depth.tolist() == [0, 0, 0, 1, 0, 1]
    status.zero_()
    # rows of no tree before and behind; a tree with more nodes than max_q says
    mask, depth = cb.tree_masks(_i32([0] * 2 + [-1, 0, -1, 0, 1, -1, 7]), q_start=_i32([2, 4, 7]), max_q=2,
                                status=status)
    assert int(status) == 5 and mask[:, 0].tolist() == [0, 0, 1, 3, 0, 0, 0, 0, 0]
    assert depth.tolist() == [0, 0, 0, 1, 0, 0, 0, 0, 0]
    status.zero_()
    mask, _ = cb.tree_masks(_i32([-1, 0, -1]), q_start=_i32([0, 2, 1]), max_q=3, status=status)
    assert int(status) == 5 and mask[:2, 0].tolist() == [1, 3]
    mask, depth = cb.tree_masks(_i32([4, 4]), q_start=_i32([1]))
    assert mask.tolist() == [[0], [0]] and depth.tolist() == [0, 0]


# ---------------------------------------------------------------- append
def rotated_64(x, cos, sin, positions):
    """(rotated, sum of the products' magnitudes)."""
    c, s = (t.double()[positions][:, None] for t in (cos, sin))
    x1, x2 = x.double()[..., 0::2], x.double()[..., 1::2]
    y = torch.cat([x1 * c - x2 * s, x1 * s + x2 * c], -1)
    return y, torch.cat([(x1 * c).abs() + (x2 * s).abs(), (x1 * s).abs() + (x2 * c).abs()], -1)


def tables(n, d, dtype):
    angle = torch.outer(torch.arange(n, device="cuda", dtype=torch.float64),
                        10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
    return angle.cos().to(dtype), angle.sin().to(dtype)


def empty_cache(kind, pages, heads, page, d, seed=0):
    g = _gen(seed)
    k, v = (torch.randn((pages, heads, page, d), device="cuda", generator=g).to(BF16) for _ in range(2))
    if kind == "bf16":
        return k, v, {}
    (k, ks), (v, vs) = quantise(k), quantise(v)
    return k, v, dict(k_scale=ks, v_scale=vs)


def held(cache, scale, slots):
    page = cache.shape[2]
    x = cache.double()[slots // page, :, slots % page]
    return x if scale is None else x * scale.double()[slots // page, :, slots % page][..., None]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("source,table", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                          (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("T,H,Hk,d,page", [(1, 4, 2, 64, 16), (37, 3, 3, 80, 32), (5, 8, 1, 16, 128),
                                           (700, 6, 2, 128, 64), (10000, 2, 1, 48, 16), (3, 1, 7, 112, 64)])
def test_append(kind, source, table, T, H, Hk, d, page):
    import computd_b200 as cb

    g = _gen(T)
    pages = -(-T // page) + 2
    k_cache, v_cache, scales = empty_cache(kind, pages, Hk, page, d)
    before = [x.clone() for x in (k_cache, v_cache, *scales.values())]
    # in place in the projection's rows
    qkv = torch.randn((T, (H + 2 * Hk) * d), device="cuda", generator=g).to(source)
    q = qkv[:, :H * d].view(T, H, d)
    k = qkv[:, H * d:(H + Hk) * d].view(T, Hk, d)
    v = qkv[:, (H + Hk) * d:].view(T, Hk, d)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    skipped = torch.arange(T, device="cuda") % 11 == 10
    slots[skipped] = -1
    cos, sin = tables(3000, d, table)
    positions = torch.randint(0, 3000, (T,), device="cuda", generator=g)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = cb.kv_cache_append(q, k, v, cos, sin, k_cache, v_cache, slots, positions=positions, status=status,
                             **scales)
    assert int(status) == 0 and got.shape == (T, H, d) and got.dtype == BF16 and got.is_contiguous()
    want, products = rotated_64(q, cos, sin, positions)
    off = (got.double() - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -22) - 2.0 ** -45 * products
    assert float(off.max()) <= 0
    kept = slots >= 0
    for x, cache, name in ((rotated_64(k, cos, sin, positions), k_cache, "k"), ((v.double(), v.double().abs()),
                                                                                v_cache, "v")):
        scale = scales.get(name + "_scale")
        want, products = x[0][kept], x[1][kept]
        tol = want.abs() * (2.0 ** -8 + 2.0 ** -22) + 2.0 ** -45 * products
        if scale is not None:
            s = scale.double()[slots[kept] // page, :, slots[kept] % page]
            exact = (want.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
            assert float(((s - exact).abs() - exact * 2.0 ** -21).max()) <= 0
            tol = want.abs() * (2.0 ** -4 + 2.0 ** -18) + (2.0 ** -10 + 2.0 ** -20) * exact[..., None]
        assert float(((held(cache, scale, slots[kept]) - want).abs() - tol).max()) <= 0
    # no other slot changed
    free = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    free[slots[kept]] = False
    for x, y in zip((k_cache, v_cache, *scales.values()), before):
        x, y = (t.view(torch.uint8) if t.dtype == E4M3 else t for t in (x, y))
        assert torch.equal(x.transpose(1, 2).flatten(0, 1)[free], y.transpose(1, 2).flatten(0, 1)[free])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T,H,d,page", [(1, 4, 64, 16), (33, 3, 80, 32), (900, 2, 128, 128)])
def test_append_in_bf16_equals_its_two_passes(kind, T, H, d, page):
    import computd_b200 as cb
    from computd_b200.lm_ops import rope_qk

    g = _gen(T)
    qkv = torch.randn((1, T, 3 * H * d), device="cuda", generator=g).to(BF16)
    qkv[0, 0, :H * d] = 1e-38  # tiny vectors, and a vector that is not finite
    qkv[0, -1, H * d:H * d + 1] = math.inf
    cos, sin = tables(T, d, BF16)
    pages = -(-T // page)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    q, k = (x.transpose(1, 2)[0] for x in rope_qk(qkv, cos, sin, H, d))
    v = qkv[0, :, 2 * H * d:].view(T, H, d)
    one, two = (empty_cache(kind, pages, H, page, d) for _ in range(2))
    cb.kv_cache_write(k, v, *one[:2], slots, **one[2])
    parts = [qkv[0, :, i * H * d:(i + 1) * H * d].view(T, H, d) for i in range(3)]
    out = torch.empty((T, H, d), dtype=BF16, device="cuda")
    got = cb.kv_cache_append(*parts, cos, sin, *two[:2], slots, q_out=out, **two[2])
    assert got is out
    bits = lambda x: x.view(torch.int16 if x.dtype == BF16 else torch.uint8 if x.dtype == E4M3 else torch.int32)  # noqa: E731
    assert torch.equal(bits(got.contiguous()), bits(q.contiguous()))
    for x, y in zip((*one[:2], *one[2].values()), (*two[:2], *two[2].values())):
        same = bits(x) == bits(y)
        if x.dtype != E4M3:  # a NaN is one whatever its bits
            same |= torch.isnan(x) & torch.isnan(y)
        assert bool(same.all())
    # without queries the same
    three = empty_cache(kind, pages, H, page, d)
    assert cb.kv_cache_append(None, *parts[1:], cos, sin, *three[:2], slots, **three[2]) is None
    assert torch.equal(bits(two[0]), bits(three[0])) and torch.equal(bits(two[1]), bits(three[1]))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T", [50, 12000])
def test_append_keeps_the_last_of_repeated_slots(kind, T):
    import computd_b200 as cb

    H, d, page, pages = 2, 32, 16, 40
    g = _gen(T)
    k, v = (torch.randn((T, H, d), device="cuda", generator=g).to(BF16) for _ in range(2))
    slots = torch.randint(0, pages * page, (T,), device="cuda", generator=g)
    cos, sin = tables(T, d, torch.float32)
    cache = empty_cache(kind, pages, H, page, d)
    cb.kv_cache_append(None, k, v, cos, sin, *cache[:2], slots, **cache[2])
    last = {}
    for t, s in enumerate(slots.tolist()):
        last[s] = t
    rows = torch.tensor(sorted(last.values()), device="cuda")
    want, _ = rotated_64(k, cos, sin, torch.arange(T, device="cuda"))
    for x, c, scale in ((want, cache[0], cache[2].get("k_scale")), (v.double(), cache[1], cache[2].get("v_scale"))):
        got = held(c, scale, slots[rows])
        amax = x[rows].abs().amax(-1, keepdim=True)
        assert float(((got - x[rows]).abs() - amax * 2.0 ** -4).max()) <= 0


def test_append_reports_positions_and_slots_outside():
    import computd_b200 as cb

    T, H, d = 6, 2, 64
    x = torch.ones((T, H, d), dtype=BF16, device="cuda")
    cos, sin = tables(4, d, torch.float32)
    for kind in ("bf16", "e4m3"):
        k, v, scales = empty_cache(kind, 2, H, 16, d)
        before = k.clone()
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        positions = torch.tensor([0, 4, -1, 3, 2 ** 40, 1], device="cuda")
        q = cb.kv_cache_append(x, x, x, cos, sin, k, v, torch.arange(T, device="cuda"), positions=positions,
                               status=status, **scales)
        assert int(status) == 5
        bad = torch.tensor([False, True, True, False, True, False], device="cuda")
        assert bool(torch.isnan(q[bad]).all()) and bool(torch.isfinite(q[~bad]).all())
        slots = torch.arange(T, device="cuda")
        assert bool(torch.isnan(held(k, scales.get("k_scale"), slots)[bad]).all())
        assert bool(torch.isfinite(held(k, scales.get("k_scale"), slots)[~bad]).all())
        assert float((held(v, scales.get("v_scale"), slots) - 1).abs().max()) <= 2.0 ** -4
        k.copy_(before)
        status.zero_()
        cb.kv_cache_append(x, x, x, cos, sin, k, v, torch.tensor([32, -2, -1, -1, 2 ** 50, -1], device="cuda"),
                           positions=positions.clamp(0, 3), status=status, **scales)
        assert int(status) == 5 and torch.equal(k.view(torch.uint8), before.view(torch.uint8))


def test_append_where_products_cancel():
    """x1 cos = x2 sin but for the last bits: the rest keeps its bits."""
    import computd_b200 as cb

    d, n = 64, 4096
    cos, sin = tables(n, d, torch.float32)
    x = torch.empty((n, 1, d), device="cuda")
    x[:, 0, 0::2], x[:, 0, 1::2] = sin, cos  # x1 c - x2 s is the tables' rounding error, or 0
    k, v, _ = empty_cache("bf16", n // 16, 1, 16, d)
    got = cb.kv_cache_append(x, x, x, cos, sin, k, v, torch.arange(n, device="cuda"))
    want, products = rotated_64(x, cos, sin, torch.arange(n, device="cuda"))
    off = (got.double() - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -22) - 2.0 ** -45 * products
    assert float(off.max()) <= 0


# ---------------------------------------------------------------- attention
def tree_attention_64(q, cache, start, seen, scale=None):
    """(out, sum p |v| / sum p) in 64 bits; seen[r]: the nodes that row r sees."""
    T, H, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((T, H, d), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b, length in enumerate(cache.lengths):
        n = start[b + 1] - start[b]
        if n == 0 or length == 0:
            continue
        k, v = cache.dense(b)
        group = H // k.shape[0]
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        rows = slice(start[b], start[b + 1])
        see = torch.zeros((n, length), dtype=torch.bool)
        prefix = length - n
        see[:, :max(prefix, 0)] = True
        for i in range(n):
            for j in seen[start[b] + i]:
                if 0 <= j < n and prefix + j >= 0:
                    see[i, prefix + j] = True
        see = see.cuda()
        used = see.any(0)  # nobody's keys and values may be anything
        k, v = torch.where(used[:, None], k, 0.0), torch.where(used[:, None], v, 0.0)
        s = torch.einsum("nhd,hld->hnl", q[rows].double(), k) * scale
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(see, torch.exp(s - top.clamp(min=-1e300)), 0.0)
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        out[rows] = torch.einsum("hnl,hld->nhd", p, v)
        mag[rows] = torch.einsum("hnl,hld->nhd", p, v.abs())
    return out, mag


def attend(cache, q, new, seen, words=None, **kw):
    import computd_b200 as cb

    words = max(1, -(-max(new) // 64)) if words is None else words
    return cb.paged_tree_attention(q, cache.k, cache.v, cache.table, cache.len, words_of(seen, words),
                                   q_start=_i32(starts(new)), max_q=max(max(new), 1), **cache.scales(), **kw)


def masks_of(new, kind, seed=0):
    rng = random.Random(seed)
    seen = []
    for n in new:
        if kind == "tree":
            seen += above(tree(n, rng, True))
        else:  # any bits, some rows none, some beyond the tree
            seen += [set() if rng.random() < 0.2 else {j for j in range(64 * max(1, -(-max(new) // 64)))
                                                       if rng.random() < 0.5} for _ in range(n)]
    return seen


# (nodes, lengths): single nodes; small trees; none, and more nodes than tokens; up to and
# beyond 64 nodes; a tree that is all there is
SHAPES = [
    ([1], [1]),
    ([1, 4, 16], [1, 4, 300]),
    ([5, 0, 7, 3], [0, 9, 3, 50]),
    ([12, 16, 1], [1000, 16, 64]),
    ([20, 33, 1], [20, 500, 64]),
    ([64, 65, 30], [1000, 65, 129]),
    ([130, 257], [200, 257]),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 4, 64, 16), (2, 2, 128, 64), (8, 2, 128, 32), (6, 1, 80, 16),
                                                   (3, 3, 16, 128), (16, 1, 48, 64), (5, 5, 112, 32)])
@pytest.mark.parametrize("new,lengths", SHAPES)
@pytest.mark.parametrize("masks", ["tree", "any"])
def test_tree_attention(kind, heads, kv_heads, d, page, new, lengths, masks):
    cache = Cache(kind, lengths, kv_heads, d, page, seed=len(new) + d)
    q = torch.randn((sum(new), heads, d), device="cuda", generator=_gen(3)).to(BF16)
    seen = masks_of(new, masks)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = attend(cache, q, new, seen, status=status)
    want, mag = tree_attention_64(q, cache, starts(new), seen)
    check(got, want, mag)
    assert int(status) == 0
    assert torch.equal(got, attend(cache, q, new, seen, words=-(-max(new) // 64) + 2))  # wider rows of bits


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,lengths", [([16] * 3, [5000, 4097, 33]), ([48, 40], [9000, 4100]),
                                         ([64] * 2, [3000, 12000]), ([200], [8192])])
def test_tree_attention_long(kind, new, lengths):
    cache = Cache(kind, lengths, 2, 128, 64, seed=1)
    q = torch.randn((sum(new), 4, 128), device="cuda", generator=_gen(4)).to(BF16)
    seen = masks_of(new, "tree", 5)
    got = attend(cache, q, new, seen)
    check(got, *tree_attention_64(q, cache, starts(new), seen))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,lengths", [([7], [40]), ([16, 3], [16, 700]), ([40], [90]), ([100], [1000])])
def test_chains_attend_as_paged_attention(kind, new, lengths):
    """A tree that is a chain is a causal chunk."""
    import computd_b200 as cb

    cache = Cache(kind, lengths, 3, 64, 16, seed=2)
    q = torch.randn((sum(new), 3, 64), device="cuda", generator=_gen(5)).to(BF16)
    seen = [set(range(i + 1)) for n in new for i in range(n)]
    got = attend(cache, q, new, seen, scale=0.2)
    want = cb.paged_attention(q, cache.k, cache.v, cache.table, cache.len, q_start=_i32(starts(new)), max_q=max(new),
                              scale=0.2, **cache.scales())
    out, mag = tree_attention_64(q, cache, starts(new), seen, 0.2)
    check(got, out, mag)
    check(want, out, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (4, 2, 128), (3, 1, 80)])
@pytest.mark.parametrize("n,length", [(5, 40), (12, 12), (33, 700), (70, 200), (140, 5000)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_a_node_may_not_see_does_not_reach_it(kind, heads, kv_heads, d, n, length, bad):
    cache = Cache(kind, [length], kv_heads, d, 16, seed=n, poison=False)
    q = torch.randn((n, heads, d), device="cuda", generator=_gen(6)).to(BF16)
    rng = random.Random(n)
    seen = masks_of([n], "any", 9)
    hidden = {rng.randrange(n) for _ in range(1 + n // 6)}
    for s in seen[:n // 2]:
        s -= hidden
    clean, mag = tree_attention_64(q, cache, [0, n], seen)
    slots = [(int(cache.table[0, (length - n + j) // 16]), (length - n + j) % 16) for j in hidden]
    channels = [1, d - 2]
    for page, off in slots:
        for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            if s is not None:
                s[page, :, off] = bad
            elif x is cache.k:
                x[page, :, off] = bad
            else:
                x[page, :, off, channels] = bad
    got = attend(cache, q, [n], seen)
    blind = torch.tensor([not (s & hidden) for s in seen], device="cuda")
    check(got[blind], clean[blind], mag[blind])
    # who sees one has keys that are not numbers, so no row of its own
    assert not bool(torch.isfinite(got[~blind]).all(-1).any())


@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (4, 2, 128), (3, 1, 80)])
@pytest.mark.parametrize("n,length", [(5, 40), (33, 700), (70, 200), (140, 5000)])
def test_values_that_are_not_finite_reach_who_sees_them(heads, kv_heads, d, n, length):
    """In their channel, and no other."""
    cache = Cache("bf16", [length], kv_heads, d, 16, seed=n, poison=False)
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
@pytest.mark.parametrize("new", [[3, 9], [40, 30], [150, 20]])
def test_tree_attention_layouts_streams_and_graphs(kind, new):
    """Strided queries, outputs and pages, rows of no sequence, another stream, a replayed graph."""
    import computd_b200 as cb

    lengths = [300, 77]
    cache = Cache(kind, lengths, 2, 64, 16, seed=8)
    for name in ("k", "v", "k_scale", "v_scale"):
        x = getattr(cache, name)
        if x is not None:  # pages twice as far apart
            wide = torch.zeros((x.shape[0], 2, *x.shape[1:]), dtype=x.dtype, device="cuda")
            wide[:, 0].copy_(x)
            setattr(cache, name, wide[:, 0])
    T, lo = sum(new) + 7, 4
    wide = torch.randn((T, 3, 4, 64), device="cuda", generator=_gen(7)).to(BF16)
    q = wide[:, 1]
    start = [lo + s for s in starts(new)]
    seen = [set()] * lo + masks_of(new, "tree", 3) + [{0}] * 3
    want, mag = tree_attention_64(q, cache, start, seen)
    mask = words_of(seen, -(-max(new) // 64))
    out = torch.full((T, 2, 4, 64), 7.0, dtype=BF16, device="cuda")
    call = lambda out: cb.paged_tree_attention(  # noqa: E731
        q, cache.k, cache.v, cache.table, cache.len, mask, q_start=_i32(start), max_q=max(new), out=out,
        **cache.scales())
    rows = slice(lo, lo + sum(new))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert call(out[:, 0]).data_ptr() == out.data_ptr()
    torch.cuda.current_stream().wait_stream(s)
    check(out[rows, 0], want[rows], mag[rows])
    assert bool((out[:lo] == 7).all()) and bool((out[rows.stop:] == 7).all()) and bool((out[:, 1] == 7).all())
    first = out[:, 0].clone()
    start_t = _i32(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cb.paged_tree_attention(q, cache.k, cache.v, cache.table, cache.len, mask, q_start=start_t, max_q=max(new),
                                out=out[:, 0], **cache.scales())
    for _ in range(2):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out[:, 0], first)


@pytest.mark.parametrize("n", [4, 40, 150])
def test_tree_attention_reports_pages_lengths_and_sizes(n):
    cache = Cache("bf16", [200, 200], 2, 64, 16, seed=3)
    q = torch.randn((2 * n, 2, 64), device="cuda", generator=_gen(8)).to(BF16)
    seen = masks_of([n, n], "tree")
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    for spoil in ("page", "length", "size"):
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        table, length = cache.table.clone(), cache.len.clone()
        max_q, starts_ = n, [0, n, 2 * n]
        if spoil == "page":
            cache.table[1, 3] = 2 ** 30
        elif spoil == "length":
            cache.len[1] = cache.table.shape[1] * 16 + 1
        else:
            max_q, starts_ = n - 1, [0, n - 1, 2 * n - 1]  # n nodes in the second
        import computd_b200 as cb
        got = cb.paged_tree_attention(q, cache.k, cache.v, cache.table, cache.len, words_of(seen, 3),
                                      q_start=_i32(starts_), max_q=max_q, status=status)
        cache.table, cache.len = table, length
        assert int(status) == 5, spoil
        rows = slice(starts_[1], starts_[2])
        assert bool(torch.isnan(got[rows]).all()), spoil
        if spoil != "size":
            check(got[:n], want[:n], mag[:n])


# ---------------------------------------------------------------- the walk
def walk_64(target, tokens, parents, u, start):
    """The rule, in 64 bits on the host."""
    B, steps = u.shape
    p = target.double().cpu()
    p = torch.where(torch.isfinite(p) & (p > 0), p, 0.0)
    kept, out, path = [], [], []
    for b in range(B):
        node, got, way = 0, [], []
        n = start[b + 1] - start[b]
        while n:
            c = torch.cumsum(p[start[b] + node], 0)
            goal = torch.tensor([float(u[b, len(got)]) * float(c[-1])], dtype=torch.float64)
            t = -1
            if float(c[-1]) > 0:
                t = int(torch.searchsorted(c, goal, right=True))
            got.append(t)
            way.append(node)
            below = [i for i in range(1, n) if parents[start[b] + i] == node and i > node
                     and tokens[start[b] + i] == t and t >= 0]
            if not below or len(got) == steps:
                break
            node = below[0]
        kept.append(max(len(got) - 1, 0))
        out.append(got + [-1] * (steps - len(got)))
        path.append(way + [-1] * (steps - len(way)))
    return kept, out, path


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 65, 2049, 32000, 64401])
@pytest.mark.parametrize("sizes,steps", [([1], 1), ([7, 0, 1, 40, 12], 4), ([100, 33], 9)])
def test_verify_tree(dtype, V, sizes, steps):
    import computd_b200 as cb

    rng = random.Random(V)
    g = _gen(V)
    trees = [tree(n, rng, True) for n in sizes]
    T = sum(sizes)
    target = torch.softmax(5 * torch.randn((T, V), device="cuda", generator=g), -1).to(dtype)
    if V > 3:  # what is no probability counts for nothing
        target[:, 2] = math.nan
        target[:, 1] = -1.0
        target[0, 0] = math.inf
    flat = [p for t in trees for p in t]
    start = starts(sizes)
    # children have their parent's likely tokens, so that walks go on
    best = target.float().nan_to_num(0, 0, 0).topk(min(3, V), -1).indices.tolist()
    tokens = [best[start[b] + max(p, 0)][rng.randrange(min(3, V))] for b, t in enumerate(trees) for p in t]
    u = torch.rand((len(sizes), steps), device="cuda", generator=g)
    u[0, 0] = 0.0
    args = (target, _i32(tokens), _i32(flat), u)
    kept, out, path = cb.verify_tree(*args, q_start=_i32(start))
    want = walk_64(target, tokens, flat, u.cpu(), start)
    assert kept.tolist() == want[0] and out.tolist() == want[1] and path.tolist() == want[2]
    assert kept.dtype == out.dtype == path.dtype == torch.int32
    for x, y in zip((kept, out, path), cb.verify_tree(*args, q_start=_i32(start))):
        assert torch.equal(x, y)


def test_verify_tree_edges():
    import computd_b200 as cb

    V = 10
    one = lambda t: torch.eye(V, device="cuda")[t]  # noqa: E731
    target = torch.stack([one(4), one(5), one(6), torch.zeros(V, device="cuda")])
    u = torch.full((1, 4), 0.5, device="cuda")
    # a chain to a row without mass
    got = cb.verify_tree(target, _i32([0, 4, 5, 6]), _i32([-1, 0, 1, 2]), u)
    assert [x.tolist() for x in got] == [[3], [[4, 5, 6, -1]], [[0, 1, 2, 3]]]
    # steps end the walk; the last token is drawn all the same
    got = cb.verify_tree(target, _i32([0, 4, 5, 6]), _i32([-1, 0, 1, 2]), u[:, :2].contiguous())
    assert [x.tolist() for x in got] == [[1], [[4, 5]], [[0, 1]]]
    # the first of two children with the token; parents that do not come before their node are none
    got = cb.verify_tree(target, _i32([0, 4, 4, 6]), _i32([-1, 0, 0, 3]), u)
    assert [x.tolist() for x in got] == [[1], [[4, 5, -1, -1]], [[0, 1, -1, -1]]]
    got = cb.verify_tree(target, _i32([4, 4, -1, 4]), _i32([0, -1, 0, 7]), u)
    assert [x.tolist() for x in got] == [[0], [[4, -1, -1, -1]], [[0, -1, -1, -1]]]
    # every uniform number gives the token whose share it falls into
    p = torch.tensor([[0.25, 0.0, 0.5, 0.25]], device="cuda").expand(5, 4).contiguous()
    u = torch.tensor([[0.0], [0.25], [0.7499], [0.75], [1 - 2.0 ** -24]], device="cuda")
    got = cb.verify_tree(p, _i32([0] * 5), _i32([-1] * 5), u)
    assert got[1].tolist() == [[0], [2], [2], [3], [3]]
    # no sequences; sequences without nodes
    none = cb.verify_tree(p[:0], _i32([]), _i32([]), u[:0], q_start=_i32([0]))
    assert [tuple(x.shape) for x in none] == [(0,), (0, 1), (0, 1)]
    none = cb.verify_tree(p[:0], _i32([]), _i32([]), u)
    assert none[0].tolist() == [0] * 5 and none[1].tolist() == none[2].tolist() == [[-1]] * 5


# ---------------------------------------------------------------- keep
def keep_plain(caches, table, start, path, kept, page):
    for x in caches:
        x = x.view(torch.uint8) if x.dtype == E4M3 else x
        old = x.clone()
        for b, n in enumerate(kept):
            for i in range(n + 1):
                a, c = start[b] + path[b][i], start[b] + i
                x[:, table[b][c // page], :, c % page] = old[:, table[b][a // page], :, a % page]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers,H,d,page,n,steps", [(1, 1, 16, 16, 5, 3), (3, 2, 80, 16, 40, 7), (2, 5, 128, 64, 64, 64),
                                                     (12, 3, 48, 32, 100, 12), (1, 2, 64, 128, 600, 300)])
def test_keep(kind, layers, H, d, page, n, steps):
    import computd_b200 as cb

    rng = random.Random(n)
    B, pages_each = 5, -(-(n + 40) // page) + 1
    g = _gen(n)
    shape = (layers, B * pages_each + 2, H, page, d)
    k, v = (torch.randn(shape, device="cuda", generator=g).to(BF16) for _ in range(2))
    scales = {}
    if kind == "e4m3":
        (k, ks), (v, vs) = quantise(k), quantise(v)
        scales = dict(k_scale=ks, v_scale=vs)
    table = torch.randperm(shape[1], device="cuda", generator=g)[:B * pages_each].view(B, pages_each).int()
    start = [rng.randrange(40) for _ in range(B)]
    kept = [0, -1, min(steps, n) - 1, rng.randrange(min(steps, n)), rng.randrange(min(steps, n))]
    path = [sorted(rng.sample(range(n), max(m, 0) + 1)) for m in kept]
    path[3] = list(range(kept[3] + 1))  # all stay
    want = [x.clone() for x in (k, v, *scales.values())]
    keep_plain(want, table.tolist(), start, path, kept, page)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    rows = _i32([p + [-1] * (steps - len(p)) for p in path])
    cb.kv_cache_keep(k, v, table, _i32(start), rows, _i32(kept), status=status, **scales)
    for x, y in zip((k, v, *scales.values()), want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert int(status) == 0
    # one layer by itself, with strided pages
    one = [x[0] for x in (k, v)]
    cb.kv_cache_keep(*one, table, _i32(start), _i32([[0] * steps] * B), _i32([0] * B), status=status,
                     **{name: x[0] for name, x in scales.items()})
    assert int(status) == 0 and torch.equal(k.view(torch.uint8), want[0].view(torch.uint8))


def test_keep_reports_bad_paths_and_pages():
    import computd_b200 as cb

    k = torch.randn((2, 12, 2, 16, 32), device="cuda", generator=_gen(0)).to(BF16)
    v = k.clone()
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(3, 4)
    good_start, good_path, good_kept = [3, 20, 0], [[0, 5, 9], [1, 2, 30], [0, 1, 7]], [2, 2, 2]
    for start, path, kept, pages in [([3, 20, 0], [[0, 5, 5]], [2, 2, 2], None),          # does not ascend
                                     ([3, 20, 0], [[-1, 5, 9]], [2, 2, 2], None),
                                     ([3, 20, 0], [[0, 5, 9]], [3, 2, 2], None),           # longer than the path
                                     ([60, 20, 0], [[0, 3, 5]], [2, 2, 2], None),          # behind the last page
                                     ([-1, 20, 0], [[0, 5, 9]], [2, 2, 2], None),
                                     ([3, 20, 0], [[0, 5, 20]], [2, 2, 2], (0, 1, 12)),
                                     ([3, 20, 0], [[0, 5, 20]], [2, 2, 2], (0, 0, -1))]:
        x, y = k.clone(), v.clone()
        want = [k.clone(), v.clone()]
        bad = table.clone()
        if pages:
            bad[pages[0], pages[1]] = pages[2]
        keep_plain(want, table.tolist(), good_start, good_path, [-1, 2, 2], 16)
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        cb.kv_cache_keep(x, y, bad, _i32(start), _i32(path + good_path[1:]), _i32(kept), status=status)
        assert int(status) == 5 and torch.equal(x, want[0]) and torch.equal(y, want[1])
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    x, y = k.clone(), v.clone()
    # what verify_tree says of a sequence without nodes; nothing stood
    cb.kv_cache_keep(x, y, table, _i32(good_start), _i32([[-1] * 3, [9, 1, 0], [-1] * 3]), _i32([0, -1, -1]),
                     status=status)
    assert int(status) == 0 and torch.equal(x, k) and torch.equal(y, v)
    assert good_kept  # the calls above differ from the good one in one place each


# ---------------------------------------------------------------- refusals
def test_tree_calls_refuse():
    import computd_b200 as cb

    k, v, _ = empty_cache("bf16", 4, 2, 16, 64)
    q = torch.zeros((6, 4, 64), dtype=BF16, device="cuda")
    kv = torch.zeros((6, 2, 64), dtype=BF16, device="cuda")
    table, lens = _i32([[0, 1], [2, 3]]), _i32([20, 20])
    mask = torch.zeros((6, 1), dtype=torch.int64, device="cuda")
    cos, sin = tables(8, 64, torch.float32)
    slots = torch.arange(6, device="cuda")
    bad = [
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask.int()),
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask[:5]),
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask[:, :0]),
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask.cpu()),
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask, max_q=65),
        lambda: cb.paged_tree_attention(q, k, v, table, lens, mask, max_q=2),
        lambda: cb.paged_tree_attention(q.float(), k, v, table, lens, mask),
        lambda: cb.paged_tree_attention(q, k, v, table.long(), lens, mask),
        lambda: cb.tree_masks(_i32([[0]])),
        lambda: cb.tree_masks(torch.zeros(3, device="cuda")),
        lambda: cb.tree_masks(_i32([-1] * 6), n_trees=4),
        lambda: cb.tree_masks(_i32([-1] * 6), n_trees=0),
        lambda: cb.tree_masks(_i32([-1] * 6), n_trees=2, q_start=_i32([0, 3, 6])),
        lambda: cb.tree_masks(_i32([-1] * 6), n_trees=2, max_q=2),
        lambda: cb.tree_masks(_i32([-1] * 5000)),
        lambda: cb.verify_tree(torch.zeros((6, 9), device="cuda").half(), _i32([0] * 6), _i32([0] * 6),
                               torch.zeros((2, 3), device="cuda")),
        lambda: cb.verify_tree(torch.zeros((6, 9), device="cuda"), _i32([0] * 5), _i32([0] * 6),
                               torch.zeros((2, 3), device="cuda")),
        lambda: cb.verify_tree(torch.zeros((6, 9), device="cuda"), _i32([0] * 6), _i32([0] * 6),
                               torch.zeros((4, 3), device="cuda")),
        lambda: cb.verify_tree(torch.zeros((6, 9), device="cuda"), _i32([0] * 6), _i32([0] * 6),
                               torch.zeros((2, 0), device="cuda")),
        lambda: cb.kv_cache_append(q[:5], kv, kv, cos, sin, k, v, slots),
        lambda: cb.kv_cache_append(q.float(), kv, kv, cos, sin, k, v, slots),
        lambda: cb.kv_cache_append(q, kv, kv, cos, sin[:7], k, v, slots),
        lambda: cb.kv_cache_append(q, kv, kv, cos.double(), sin.double(), k, v, slots),
        lambda: cb.kv_cache_append(q, kv, kv, cos[:5], sin[:5], k, v, slots),
        lambda: cb.kv_cache_append(q, kv, kv, cos[:, :30], sin[:, :30], k, v, slots),
        lambda: cb.kv_cache_append(q, kv, kv, cos, sin, k, v, slots, positions=slots.int()),
        lambda: cb.kv_cache_append(q, kv, kv, cos, sin, k, v, slots, q_out=q[:5]),
        lambda: cb.kv_cache_append(None, kv, kv, cos, sin, k, v, slots, q_out=q),
        lambda: cb.kv_cache_append(q, kv, kv, cos, sin, k, v, slots, k_scale=cos, v_scale=cos),
        lambda: cb.kv_cache_keep(k, v, table, lens, _i32([0, 0]), lens),
        lambda: cb.kv_cache_keep(k, v, table, lens, _i32([[0], [0]]), _i32([0])),
        lambda: cb.kv_cache_keep(k, v[:3], table, lens, _i32([[0], [0]]), lens),
        lambda: cb.kv_cache_keep(k[None], v, table, lens, _i32([[0], [0]]), lens),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(TypeError):
        cb.tree_masks([0])
    with pytest.raises(ValueError, match="grad"):
        cb.kv_cache_append(q, kv, kv, cos.clone().requires_grad_(), sin, k, v, slots)


# ---------------------------------------------------------------- a run of them together
def _model(r, dh):
    from test_gpu_lm_extend import _model

    return _model(r, dh)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("r,dh", [(0, 32), (2, 16)])
def test_verify_tree_step(dtype, r, dh):
    """A step's decisions are the 64-bit walk's on the probabilities of its extend; the path's tokens
    stand at their places in the cache, and the next step goes on from there."""
    import copy

    cfg, model = _model(r, dh)
    g = _gen(5)
    B, N, steps = 3, 9, 4
    cache = model.new_cache(24, page_size=16, dtype=dtype)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(2))[:15].view(B, 5).int().cuda()
    prompt = torch.randint(0, cfg.vocab, (B, 20), device="cuda", generator=g)
    lengths = _i32([20] * B)
    last = model.extend(prompt.reshape(-1), cache, table, lengths).view(B, 20, -1)[:, -1].argmax(-1)
    rng = random.Random(1)
    for _ in range(3):
        parents = [[rng.randrange(i) for i in range(1, N + 1)] for _ in range(B)]
        parents[1][-1] = -1  # no such draft
        drafts = torch.randint(0, cfg.vocab, (B, N), device="cuda", generator=g).int()
        drafts[2, 3] = cfg.vocab + 7
        u = torch.rand((B, steps), device="cuda", generator=g)
        # children of the root get the drawn token at times, so that paths are kept
        par = [p for row in parents for p in [-1] + row]
        chunk = torch.cat([last.int()[:, None], drafts], 1)
        trial = copy.deepcopy(cache)
        logits = model.extend(chunk.reshape(-1).clamp(0, cfg.vocab - 1).long(), trial, table, lengths + N + 1,
                              parents=_i32(par))
        probs = torch.softmax(logits.float(), -1)
        for b in range(B):
            c = probs[b * (N + 1)].double().cumsum(-1)
            t = int((c <= float(u[b, 0]) * c[-1]).sum())
            child = parents[b].index(0) if 0 in parents[b] else 0
            if b != 1:
                drafts[b, child] = t
        chunk = torch.cat([last.int()[:, None], drafts], 1)
        trial = copy.deepcopy(cache)
        logits = model.extend(chunk.reshape(-1).clamp(0, cfg.vocab - 1).long(), trial, table, lengths + N + 1,
                              parents=_i32(par))
        probs = torch.softmax(logits.float(), -1)
        want = walk_64(probs, chunk.reshape(-1).tolist(), par, u.cpu(), starts([N + 1] * B))
        accepted, tokens, new = model.verify_tree(last, drafts, _i32(parents), u, cache, table, lengths)
        assert accepted.tolist() == want[0] and tokens.tolist() == want[1]
        assert new.tolist() == [int(n) + 1 + a for n, a in zip(lengths, want[0])]
        # the kept tokens in the tree's chunk, at their places
        for b in range(B):
            for i, node in enumerate(want[2][b][:want[0][b] + 1]):
                at, frm = int(lengths[b]) + i, int(lengths[b]) + node
                for x, y in ((cache.k, trial.k), (cache.v, trial.v), (cache.k_scale, trial.k_scale),
                             (cache.v_scale, trial.v_scale)):
                    if x is not None:
                        assert torch.equal(x[:, table[b, at // 16].long(), :, at % 16].float(),
                                           y[:, table[b, frm // 16].long(), :, frm % 16].float())
        last = tokens[torch.arange(B), accepted.long()]
        lengths = new
    cache.check()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_tree_logits_are_the_paths_logits(dtype):
    """Behind every node stand the logits of its path as a chunk of its own, up to the roundings
    of another kernel and order: the differences are of the size of bf16 activations' steps."""
    cfg, model = _model(0, 32)
    B, n = 3, 7
    parents = [-1, 0, 0, 1, 1, 2, 5]
    cache, plain = (model.new_cache(24, page_size=16, dtype=dtype) for _ in range(2))
    table = torch.arange(15, device="cuda", dtype=torch.int32).view(B, 5)
    g = _gen(6)
    prompt = torch.randint(0, cfg.vocab, (B, 18), device="cuda", generator=g)
    nodes = torch.randint(0, cfg.vocab, (B, n), device="cuda", generator=g)
    for c in (cache, plain):
        model.extend(prompt.reshape(-1), c, table, _i32([18] * B))
    logits = model.extend(nodes.reshape(-1), cache, table, _i32([18 + n] * B),
                          parents=_i32(parents * B)).view(B, n, -1).float()
    for path in ([0, 1, 3], [0, 1, 4], [0, 2, 5, 6]):
        chain = model.extend(nodes[:, path].reshape(-1), plain, table,
                             _i32([18 + len(path)] * B)).view(B, len(path), -1).float()
        # every block's keys at a node are its path's: layer 0 exactly
        for i, node in enumerate(path):
            for b in range(B):
                a, c = 18 + node, 18 + i
                assert torch.equal(cache.k[0, table[b, a // 16].long(), :, a % 16].view(torch.uint8),
                                   plain.k[0, table[b, c // 16].long(), :, c % 16].view(torch.uint8))
        diff = (logits[:, path] - chain).abs().amax()
        assert float(diff) <= 0.05 * float(chain.abs().amax()), float(diff)
    cache.check()


def test_verify_tree_reports_last_tokens_outside_the_vocabulary():
    import computd_b200 as cb

    cfg, model = _model(0, 32)
    cache = model.new_cache(24, page_size=16)
    table = torch.arange(15, device="cuda", dtype=torch.int32).view(3, 5)
    lengths = _i32([0, 4, 9])
    model.extend(torch.zeros(27, dtype=torch.long, device="cuda"), cache, table, _i32([9] * 3))
    accepted, tokens, new = model.verify_tree(_i32([1, -1, cfg.vocab]), _i32([[3, 4]] * 3), _i32([0, 1]),
                                              torch.rand((3, 3), device="cuda", generator=_gen(1)), cache, table, lengths)
    assert accepted[1:].tolist() == [0, 0] and tokens[1:].tolist() == [[-1] * 3] * 2 and new[1:].tolist() == [4, 9]
    assert int(tokens[0, 0]) >= 0
    with pytest.raises(cb.DWAError):
        cache.check()
