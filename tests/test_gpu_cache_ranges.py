"""GPU: attention over e4m3 caches whose tokens are of very different sizes.

A key or a value that a row may not see must not change that row, however large it is,
nor may one that it sees without weight.  Bounds as in test_gpu_decode.py: every
rounding there is relative to a row's own weights, or to one token's own scale.
"""
import math

import pytest
import torch

from test_gpu_decode import Cache, attend, attention_64, check, starts

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _at(cache, b, token):
    return cache.table[b, token // cache.page].long(), token % cache.page


def _queries(n, heads, d, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, heads, d), device="cuda", generator=g).to(BF16)


# (new tokens, heads, heads of the cache): a few rows per head, two column tiles of them, many
FORMS = [(2, 4, 2), (9, 2, 2), (140, 2, 2)]


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("d,page", [(64, 16), (80, 32), (128, 64)])
@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("log2", [11, 27, 40, 100])
def test_hidden_tokens_of_any_size(new, heads, kv_heads, d, page, what, log2):
    """The last new token's scales are 2^log2 times what they were: the rows before it are as
    exact as without it.  (Its own row has a key whose score is +-2^log2, or its value's.)"""
    lengths = [new + 200, new]
    cache = Cache("e4m3", lengths, kv_heads, d, page, seed=d + new)
    q = _queries(2 * new, heads, d, seed=log2)
    for b in range(2):
        at = _at(cache, b, lengths[b] - 1)
        for name in ("k", "v") if what == "both" else (what,):
            scale = cache.k_scale if name == "k" else cache.v_scale
            scale[at[0], :, at[1]] *= 2.0 ** log2
    want, mag = attention_64(q, cache, starts([new, new]))
    got = attend(cache, q, [new, new])
    if what != "v":  # scores of 2^100 are beyond what the last rows are asked for
        keep = torch.ones(2 * new, dtype=torch.bool, device="cuda")
        keep[[new - 1, 2 * new - 1]] = log2 < 40
        got, want, mag = got[keep], want[keep], mag[keep]
    check(got, want, mag)


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", [0, 60, 333])
@pytest.mark.parametrize("log2", [11, 40, 100])
def test_visible_tokens_without_weight(new, heads, kv_heads, d, where, log2):
    """A cached token whose scores are far below every other's, with a value 2^log2 times
    larger: its weight, below 2^-800, leaves nothing of it."""
    lengths = [new + 400]
    cache = Cache("e4m3", lengths, kv_heads, d, 32, seed=d + new)
    q = (_queries(new, heads, d, seed=log2).abs() + 0.5).to(BF16)
    at = _at(cache, 0, where)
    cache.k[at[0], :, at[1]] = torch.full((d,), -448.0, device="cuda").to(cache.k.dtype)
    cache.k_scale[at[0], :, at[1]] = 1.0  # a score of -448 sum q / sqrt(d), below -2800
    cache.v_scale[at[0], :, at[1]] *= 2.0 ** log2
    want, mag = attention_64(q, cache, [0, new])
    check(attend(cache, q, [new]), want, mag)
    # and a key so much larger than all others
    cache.k_scale[at[0], :, at[1]] = 2.0 ** log2
    check(attend(cache, q, [new]), want, mag)


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("log2", [-118, -100, 100, 116])
def test_all_values_small_or_large(new, heads, kv_heads, log2):
    """Values from 2^-116 on (the smallest scale is 2^-126), and up to 2^118."""
    lengths = [new + 300, new + 1]
    cache = Cache("e4m3", lengths, kv_heads, 128, 32, seed=new)
    q = _queries(2 * new, heads, 128, seed=3)
    cache.v_scale *= 2.0 ** log2
    want, mag = attention_64(q, cache, starts([new, new]))
    got = attend(cache, q, [new, new])
    check((got.double() * 2.0 ** -log2), want * 2.0 ** -log2, mag * 2.0 ** -log2)


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
def test_zero_vectors_among_others(new, heads, kv_heads):
    """Zero keys and values have the scale 2^-126: seen or not, at the start, in the middle and
    behind everything."""
    lengths = [new + 300, new]
    cache = Cache("e4m3", lengths, kv_heads, 64, 16, seed=new)
    for b, length in enumerate(lengths):
        for token in (0, length // 2, length - 1):
            at = _at(cache, b, token)
            for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                codes.view(torch.uint8)[at[0], :, at[1]] = 0
                scale[at[0], :, at[1]] = 2.0 ** -126
    q = _queries(2 * new, heads, 64, seed=1)
    want, mag = attention_64(q, cache, starts([new, new]))
    check(attend(cache, q, [new, new]), want, mag)


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("length", [600, 9000])
def test_scales_all_over_the_range(new, heads, kv_heads, length):
    """Value scales of 2^-100 to 2^100 from one token to the next, one sequence alone (its
    context is split) and two of very different lengths."""
    g = torch.Generator(device="cuda").manual_seed(length + new)
    cache = Cache("e4m3", [length, new + 2], kv_heads, 128, 64, seed=4, poison=False)
    cache.v_scale *= torch.exp2(200 * torch.rand(cache.v_scale.shape, device="cuda", generator=g) - 100)
    q = _queries(2 * new, heads, 128, seed=9)
    want, mag = attention_64(q, cache, starts([new, new]))
    check(attend(cache, q, [new, new]), want, mag)


@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("what", ["k", "v"])
def test_hidden_scales_that_are_not_finite(new, heads, kv_heads, bad, what):
    """The last new token's scale is no number: that token's row is none, the others are exact."""
    lengths = [new + 100]
    cache = Cache("e4m3", lengths, kv_heads, 128, 32, seed=new)
    q = _queries(new, heads, 128, seed=5)
    want, mag = attention_64(q, cache, [0, new])
    at = _at(cache, 0, lengths[0] - 1)
    (cache.k_scale if what == "k" else cache.v_scale)[at[0], :, at[1]] = bad
    got = attend(cache, q, [new])
    check(got[:-1], want[:-1], mag[:-1])
    if what == "v":
        assert not bool(torch.isfinite(got[-1]).any())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("length", [0, 1000])
@pytest.mark.parametrize("new,heads,kv_heads", FORMS)
@pytest.mark.parametrize("log2", [20, 23, 27, 60])
def test_large_scores(new, heads, kv_heads, log2, length, kind):
    """Scores of 2^log2 and more, whose steps in f32 are a good part of 1: the outputs are those
    of one key each, with no error but its value's and the result's rounding.  (1000 keys more:
    over several blocks.)"""
    lengths = [new + 120 + length]
    cache = Cache(kind, lengths, kv_heads, 64, 32, seed=new)
    if kind == "e4m3":
        cache.v_scale *= torch.exp2(torch.arange(32, device="cuda") % 7 - 3.0)
    q = (_queries(new, heads, 64, seed=6).float() * 2.0 ** log2).to(BF16)
    # only rows with a clear winner: by 2^-8 of the largest score, far beyond the sums' error
    k, _ = cache.dense(0)
    s = torch.einsum("nhd,hld->nhl", q.double(), k.repeat_interleave(heads // kv_heads, 0)) / 8
    see = torch.arange(lengths[0], device="cuda") < (lengths[0] - new + 1 + torch.arange(new, device="cuda"))[:, None]
    top = s.masked_fill(~see[:, None], -math.inf).topk(2, -1).values
    clear = top[..., 0] - top[..., 1] > 2.0 ** -8 * s.abs().amax(-1)
    assert float(clear.float().mean()) > 0.7
    want, mag = attention_64(q, cache, [0, new])
    got = attend(cache, q, [new])
    check(got[clear], want[clear], mag[clear])
