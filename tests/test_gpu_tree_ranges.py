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
    "few": (12, 4, 2, 400),
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
