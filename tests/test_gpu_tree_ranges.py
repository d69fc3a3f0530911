"""GPU: attention of a tree's nodes over caches whose scores, keys or values are far apart, in every kernel that
the call may pick; bounds as in test_gpu_decode.py (every rounding there is relative to a row's own
weights, or to one token's own scale) and test_gpu_tree_batches.py.
"""
import math

import pytest
import torch
from test_gpu_decode import BF16, Cache, check, starts
from test_gpu_draft_trees import _gen, attend, masks_of, tree_attention_64

pytestmark = pytest.mark.gpu

# (nodes, heads, heads of the cache, tokens): up to 16 rows per head; 17 to 32 with a block to a unit, with keys
# shared among blocks, with two blocks to an SM and of one step; 33 to 64 with a block to 32 rows, with two
# blocks to an SM and over long contexts; more
FORMS = {
    "few": (8, 4, 2, 400),
    "pairs": (12, 4, 2, 400),
    "whole": (24, 2, 2, 600),
    "grouped": (8, 8, 2, 600),
    "shared": (32, 2, 2, 2500),
    "short": (17, 160, 160, 300),
    "one_step": (20, 2, 2, 90),
    "room": (48, 2, 2, 700),
    "short_two": (48, 96, 96, 300),
    "long_two": (64, 2, 2, 2500),
    "many": (140, 2, 2, 500),
}
forms = pytest.mark.parametrize("form", list(FORMS))


def _queries(n, heads, d, seed):
    return torch.randn((n, heads, d), device="cuda", generator=_gen(seed)).to(BF16)


def _at(cache, b, token):
    return cache.table[b, token // cache.page].long(), token % cache.page


def _tokens(cache, b, tokens):
    """Pages and places of a sequence's tokens, as an index."""
    tokens = torch.as_tensor(tokens, device="cuda")
    return cache.table[b][tokens // cache.page].long(), tokens % cache.page


@forms
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("masks", ["tree", "any"])
def test_scale_zero(form, kind, masks):
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache(kind, [length, n], kv_heads, 64, 16, seed=2)
    q, seen = _queries(2 * n, heads, 64, 1), masks_of([n, n], masks, 3)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen, scale=0.0)
    check(attend(cache, q, [n, n], seen, scale=0.0), want, mag)


@forms
@pytest.mark.parametrize("how", ["keys", "products"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [1, 128, 260])
def test_scores_of_minus_infinity(form, how, d, first):
    """The first cached tokens' scores, whose weight is 0 beside any other; with all of them a row has
    nothing to see and gets zeros.  (Products: sums of them beyond f32.)"""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache("bf16", [length], kv_heads, d, 16, seed=2, poison=False)
    q, seen = _queries(n, heads, d, 4).abs() + 0.25, masks_of([n], "any", 3)
    q, scale = (q.to(BF16), None) if how == "keys" else ((q * 2.0 ** 60).to(BF16), 2.0 ** -63)
    for count in (min(first, length), length):
        at = _tokens(cache, 0, list(range(count)))
        cache.k[at[0], :, at[1]] = -math.inf
        want, mag = tree_attention_64(q, cache, [0, n], seen, scale=scale)
        if count == length:
            assert not want.any()
        if how == "products":
            cache.k[at[0], :, at[1]] = -3e38
        check(attend(cache, q, [n], seen, scale=scale), want, mag)


@pytest.mark.parametrize("form", [f for f in FORMS if f not in ("long_two", "many")])
@pytest.mark.parametrize("first", [1, 128, 260])
def test_scales_of_infinity(form, first):
    """Negative codes times an infinite scale, where scores are formed from codes.  (The kernel of many rows
    forms keys first, to which such a scale is NaN; what writes the cache makes none.)"""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache("e4m3", [length], kv_heads, 128, 16, seed=2, poison=False)
    q, seen = (_queries(n, heads, 128, 4).abs() + 0.25).to(BF16), masks_of([n], "any", 3)
    for count in (min(first, length), length):
        page, off = _tokens(cache, 0, list(range(count)))
        cache.k[page, :, off] = torch.full((), -1.0, device="cuda").to(cache.k.dtype)
        cache.k_scale[page, :, off] = math.inf
        want, mag = tree_attention_64(q, cache, [0, n], seen)
        if count == length:
            assert not want.any()
        check(attend(cache, q, [n], seen), want, mag)


def _pair(form, kind, d, page, seed, poison=True):
    """Two sequences of a form, the second of nothing but its tree."""
    n, heads, kv_heads, length = FORMS[form]
    return n, heads, Cache(kind, [length, n], kv_heads, d, page, seed=seed, poison=poison)


@forms
@pytest.mark.parametrize("d,page", [(64, 16), (80, 32), (128, 64)])
@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("log2", [11, 27, 40, 100])
def test_hidden_tokens_of_any_size(form, d, page, what, log2):
    """A leaf's scales are 2^log2 times what they were: the other nodes' rows are as exact as without it.  (Its
    own row has a key whose score is +-2^log2, or its value's.)"""
    n, heads, cache = _pair(form, "e4m3", d, page, d)
    q, seen = _queries(2 * n, heads, d, log2), masks_of([n, n], "tree", 7)
    for b in range(2):
        leaf = n // 2 if b else n - 1
        for r, nodes in enumerate(seen[b * n:(b + 1) * n]):
            if r != leaf:
                nodes.discard(leaf)  # whatever was below it
        at = _at(cache, b, cache.lengths[b] - n + leaf)
        for name in ("k", "v") if what == "both" else (what,):
            scale = cache.k_scale if name == "k" else cache.v_scale
            scale[at[0], :, at[1]] *= 2.0 ** log2
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    got = attend(cache, q, [n, n], seen)
    if what != "v":  # scores of 2^100 are beyond what the leaves' rows are asked for
        keep = torch.ones(2 * n, dtype=torch.bool, device="cuda")
        keep[[n - 1, n + n // 2]] = log2 < 40
        got, want, mag = got[keep], want[keep], mag[keep]
    check(got, want, mag)


@forms
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", [0, 37, -1])
@pytest.mark.parametrize("log2", [11, 40, 100])
def test_visible_tokens_without_weight(form, d, where, log2):
    """A cached token before the tree whose scores are far below every other's, with a value 2^log2 times
    larger: its weight, below 2^-800, leaves nothing of it."""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache("e4m3", [length], kv_heads, d, 32, seed=d + n)
    q, seen = (_queries(n, heads, d, log2).abs() + 0.5).to(BF16), masks_of([n], "any", 2)
    at = _at(cache, 0, where % (length - n))
    cache.k[at[0], :, at[1]] = torch.full((d,), -448.0, device="cuda").to(cache.k.dtype)
    cache.k_scale[at[0], :, at[1]] = 1.0  # a score of -448 sum q / sqrt(d), below -2800
    cache.v_scale[at[0], :, at[1]] *= 2.0 ** log2
    want, mag = tree_attention_64(q, cache, [0, n], seen)
    check(attend(cache, q, [n], seen), want, mag)
    # and a key so much larger than all others
    cache.k_scale[at[0], :, at[1]] = 2.0 ** log2
    check(attend(cache, q, [n], seen), want, mag)


@forms
@pytest.mark.parametrize("log2", [-118, -100, 100, 116])
def test_all_values_small_or_large(form, log2):
    """Values from 2^-116 on (the smallest scale is 2^-126), and up to 2^118."""
    n, heads, cache = _pair(form, "e4m3", 128, 32, 4)
    q, seen = _queries(2 * n, heads, 128, 3), masks_of([n, n], "tree", 3)
    cache.v_scale *= 2.0 ** log2
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    got = attend(cache, q, [n, n], seen)
    # a result below 2^-126, where bf16's step is 2^-133, is off by half of that
    off = (got.double() - want).abs() - (2.0 ** -8 + 2.0 ** -11) * mag - 2.0 ** -8 * want.abs() - 2.0 ** -134
    assert float((off * 2.0 ** -log2).max()) <= 0


@forms
def test_zero_vectors_among_others(form):
    """Zero keys and values have the scale 2^-126: seen or not, at the start, in the middle and in the tree."""
    n, heads, cache = _pair(form, "e4m3", 64, 16, 5)
    for b, length in enumerate(cache.lengths):
        for token in (0, length // 2, length - 1):
            at = _at(cache, b, token)
            for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                codes.view(torch.uint8)[at[0], :, at[1]] = 0
                scale[at[0], :, at[1]] = 2.0 ** -126
    q, seen = _queries(2 * n, heads, 64, 1), masks_of([n, n], "any", 1)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    check(attend(cache, q, [n, n], seen), want, mag)


def _least_weights(q, cache, start, seen):
    """What the rounding of a row's smallest weights may leave in its outputs.  A weight times its value's scale,
    p_j s_j, becomes fp16 in units in which the row's largest is 2^6 or more (so that everything down to 2^-20 of
    it has 11 bits); below fp16's normal numbers it is off by half of their step, 2^-25, which is 2^-31 of the largest.
    An output takes it times the value's code: 2^-31 max_j p_j s_j sum_j |code_j|."""
    T, H, d = q.shape
    out = torch.zeros((T, H, d), dtype=torch.float64, device="cuda")
    for b, length in enumerate(cache.lengths):
        n = start[b + 1] - start[b]
        (k, v), group = cache.dense(b), H // cache.k.shape[1]
        page, off = _tokens(cache, b, list(range(length)))
        scale = cache.v_scale[page, :, off].double().t().repeat_interleave(group, 0)
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        see = torch.ones((n, length), dtype=torch.bool)
        see[:, length - n:] = torch.tensor([[j in s for j in range(n)] for s in seen[start[b]:start[b + 1]]])
        s = torch.einsum("nhd,hld->hnl", q[start[b]:start[b + 1]].double(), k) * d ** -0.5
        p = torch.softmax(s.masked_fill(~see.cuda(), -math.inf), -1).nan_to_num(0.0)
        most = (p * scale[:, None]).amax(-1)
        codes = torch.einsum("nl,hld->hnd", see.cuda().double(), v.abs() / scale[..., None])
        out[start[b]:start[b + 1]] = (2.0 ** -31 * most[..., None] * codes).transpose(0, 1)
    return out


@forms
@pytest.mark.parametrize("masks", ["tree", "any"])
@pytest.mark.parametrize("whole", [False, True])
def test_scales_all_over_the_range(form, masks, whole):
    """Value scales of 2^-100 to 2^100 from one token to the next; or all alike before the tree and all over the
    range in it."""
    n, heads, cache = _pair(form, "e4m3", 128, 64, 4, poison=False)
    scale = cache.v_scale.clone()
    cache.v_scale *= torch.exp2(200 * torch.rand(cache.v_scale.shape, device="cuda", generator=_gen(n)) - 100)
    if not whole:
        at = _tokens(cache, 0, list(range(cache.lengths[0] - n)))
        cache.v_scale[at[0], :, at[1]] = scale[at[0], :, at[1]]
    q, seen = _queries(2 * n, heads, 128, 9), masks_of([n, n], masks, 5)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    got = attend(cache, q, [n, n], seen)
    tol = (2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -8 * want.abs() + _least_weights(q, cache, [0, n, 2 * n], seen)
    assert bool(torch.isfinite(got).all()) and float(((got.double() - want).abs() - tol).max()) <= 0


@forms
@pytest.mark.parametrize("shared", [0, 1])
def test_scales_that_part_ways_late(form, shared):
    """The first tiles' values are alike, then their scales rise, or fall, by 2^120."""
    n, heads, cache = _pair(form, "e4m3", 128, 64, 4, poison=False)
    length = cache.lengths[0]
    at = _tokens(cache, 0, list(range(length // 2, length)))
    cache.v_scale *= 2.0 ** (-60 if shared else 58)
    cache.v_scale[at[0], :, at[1]] *= 2.0 ** (120 if shared else -120)
    q, seen = _queries(2 * n, heads, 128, 9), masks_of([n, n], "tree", 5)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    check(attend(cache, q, [n, n], seen), want, mag)


@forms
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("log2", [18, 20, 23, 27, 29, 31, 33, 60])
@pytest.mark.parametrize("late", [False, True])
def test_large_scores(form, log2, kind, late):
    """Scores of 2^log2 and more, whose steps in f32 are a good part of 1: the outputs are those of one key each,
    with no error but its value's and the result's rounding.  (late: the keys of the first half are 2^-20 of the
    others, so that large scores come behind small ones.)"""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache(kind, [length], kv_heads, 64, 32, seed=n)
    if kind == "e4m3":
        cache.v_scale *= torch.exp2(torch.arange(32, device="cuda") % 7 - 3.0)
    if late:
        page, off = _tokens(cache, 0, list(range(length // 2)))
        if kind == "e4m3":
            cache.k_scale[page, :, off] *= 2.0 ** -20
        else:
            cache.k[page, :, off] = (cache.k[page, :, off].float() * 2.0 ** -20).to(BF16)
    q = (_queries(n, heads, 64, 6).float() * 2.0 ** log2).to(BF16)
    seen = masks_of([n], "tree", 6)
    # only rows with a clear winner: by 2^-8 of the largest score, far beyond the sums' error
    k, _ = cache.dense(0)
    s = torch.einsum("nhd,hld->nhl", q.double(), k.repeat_interleave(heads // kv_heads, 0)) / 8
    see = torch.ones((n, length), dtype=torch.bool)
    see[:, length - n:] = torch.tensor([[j in nodes for j in range(n)] for nodes in seen])
    s = s.masked_fill(~see.cuda()[:, None], -math.inf)
    top = s.topk(2, -1).values
    clear = top[..., 0] - top[..., 1] > 2.0 ** -8 * s.masked_fill(~see.cuda()[:, None], 0).abs().amax(-1)
    assert float(clear.float().mean()) > 0.7
    want, mag = tree_attention_64(q, cache, [0, n], seen)
    got = attend(cache, q, [n], seen)
    check(got[clear], want[clear], mag[clear])


@forms
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("sign", [-1, 1])
def test_large_scores_of_one_size(form, kind, sign):
    """All of a row's scores are the same number of 2^30 and more, of either sign: its output is the values' mean."""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache(kind, [length], kv_heads, 64, 32, seed=n)
    cache.k[:] = torch.ones((), device="cuda").to(cache.k.dtype)
    if kind == "e4m3":
        cache.k_scale[:] = 1.0
    q = torch.full((n, heads, 64), sign * 1.0 * 2.0 ** 28, device="cuda")
    q = (q * (1 + torch.arange(n, device="cuda") % 4)[:, None, None]).to(BF16)
    seen = masks_of([n], "tree", 6)
    want, mag = tree_attention_64(q, cache, [0, n], seen)
    check(attend(cache, q, [n], seen), want, mag)


@forms
def test_tiny_queries_and_large_keys(form):
    """Rows of q down to bf16's subnormal numbers against keys whose scales make up for it."""
    n, heads, cache = _pair(form, "e4m3", 128, 64, 6, poison=False)
    cache.k_scale = cache.k_scale * 2.0 ** 120
    q = _queries(2 * n, heads, 128, n).float()
    q = (q * torch.exp2(torch.randint(-128, -122, (2 * n, 1, 1), device="cuda", generator=_gen(n)).float())).to(BF16)
    seen = masks_of([n, n], "any", 6)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen, scale=1.0)
    check(attend(cache, q, [n, n], seen, scale=1.0), want, mag)


@forms
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_sizes_far_apart(form, kind):
    """Values from 2^-24 to 2^24 and keys from 2^-16 to 1 from one token to the next, rows of q from 2^-100 to 1;
    then scores of 2^20 and more: one key takes all, and nothing but numbers comes out."""
    n, heads, cache = _pair(form, kind, 128, 32, 21, poison=False)
    g = _gen(n)
    pages = cache.k.shape[0]
    kf = torch.exp2(torch.randint(-16, 1, (pages, 1, 32, 1), device="cuda", generator=g).float())
    vf = torch.exp2(torch.randint(-24, 25, (pages, 1, 32, 1), device="cuda", generator=g).float())
    if kind == "bf16":
        cache.k, cache.v = (cache.k.float() * kf).to(BF16), (cache.v.float() * vf).to(BF16)
    else:
        cache.k_scale, cache.v_scale = cache.k_scale * kf[..., 0], cache.v_scale * vf[..., 0]
    q = torch.randn((2 * n, heads, 128), device="cuda", generator=g)
    q = (q * torch.exp2(torch.randint(-100, 1, (2 * n, 1, 1), device="cuda", generator=g).float())).to(BF16)
    seen = masks_of([n, n], "any", 8)
    want, mag = tree_attention_64(q, cache, [0, n, 2 * n], seen)
    check(attend(cache, q, [n, n], seen), want, mag)
    big = (q.float().sign() * 2.0 ** 20).to(BF16)
    assert bool(torch.isfinite(attend(cache, big, [n, n], seen)).all())


@forms
@pytest.mark.parametrize("log2", [-100, 60, 100])
def test_large_values_behind_rising_scores(form, log2):
    """bf16 values of any size, with scores that rise by 50 (in powers of two) along the context: what weights
    are relative to moves with them, and sums stay in f32's range."""
    n, heads, kv_heads, length = FORMS[form]
    cache = Cache("bf16", [length], kv_heads, 64, 32, seed=n)
    page, off = _tokens(cache, 0, list(range(length)))
    rise = torch.arange(length, device="cuda") / length * 50 * math.log(2)  # q's first channel is 8, the scale 1/8
    cache.k[page, :, off] = (cache.k[page, :, off].float() / 16).to(BF16)
    cache.k[page, :, off, 0] = rise[:, None].to(BF16).expand(-1, kv_heads)
    cache.v[page, :, off] = (cache.v[page, :, off].float() * 2.0 ** log2).to(BF16)
    q = _queries(n, heads, 64, 3)
    q[..., 0] = 8.0
    seen = masks_of([n], "tree", 6)
    want, mag = tree_attention_64(q, cache, [0, n], seen)
    got = attend(cache, q, [n], seen)
    assert bool(torch.isfinite(got).all())
    check(got.double() * 2.0 ** -log2, want * 2.0 ** -log2, mag * 2.0 ** -log2)
