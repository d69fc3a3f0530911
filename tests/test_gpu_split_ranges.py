"""GPU: attention of many rows over a context that several blocks share, with e4m3 values near the ends of
f32's range; bounds as in test_gpu_decode.py, and half of bf16's least step, 2^-134, for what is below its normal
numbers.
"""
import pytest
import torch
from test_gpu_decode import BF16, Cache, attend, attention_64, starts
from test_gpu_draft_trees import _gen, masks_of, tree_attention_64
from test_gpu_draft_trees import attend as attend_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,lengths", [(70, [2500]), (300, [9000, 400]), (64, [5000, 3000, 70])])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("log2", [-118, -100, 100, 116])
def test_values_of_shared_contexts(causal, n, lengths, d, log2):
    cache = Cache("e4m3", lengths, 2, d, 64, seed=n)
    cache.v_scale *= 2.0 ** log2
    new = [n] * len(lengths)
    q = torch.randn((sum(new), 2, d), device="cuda", generator=_gen(n)).to(BF16)
    if causal:
        want, mag = attention_64(q, cache, starts(new))
        got = attend(cache, q, new)
    else:
        seen = masks_of(new, "tree", 3)
        want, mag = tree_attention_64(q, cache, starts(new), seen)
        got = attend_tree(cache, q, new, seen)
    tol = (2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -8 * want.abs() + 2.0 ** -134
    assert bool(torch.isfinite(got).all())
    assert float((((got.double() - want).abs() - tol) * 2.0 ** -log2).max()) <= 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("log2", [-60, 60])
def test_parts_whose_values_differ(causal, log2):
    """One half of the context has values 2^log2 times the other's, and scores that make up for it."""
    n, length = 80, 4096
    cache = Cache("e4m3", [length], 2, 128, 64, seed=5, poison=False)
    page = cache.table[0, :length // 128].long()
    cache.v_scale[page] *= 2.0 ** log2
    q = torch.randn((n, 2, 128), device="cuda", generator=_gen(n)).to(BF16)
    q[..., 0] = 16.0
    codes = torch.full((), 1.0, device="cuda").to(cache.k.dtype)
    cache.k[..., 0] = codes  # a code of 1 for all, scaled to what makes up for it
    cache.k_scale[:] = 1.0
    cache.k[..., 1:].view(torch.uint8)[:] = 0
    shift = -log2 * 0.6931471805599453 * 128 ** 0.5 / 16.0
    cache.k_scale[page] = 1.0 + shift  # negative where scores fall
    seen = masks_of([n], "tree", 3)
    want, mag = attention_64(q, cache, [0, n]) if causal else tree_attention_64(q, cache, [0, n], seen)
    got = attend(cache, q, [n]) if causal else attend_tree(cache, q, [n], seen)
    # keys are rounded to 2^-12: the scores, of up to 70 in natural units, move by 2^-6 at most, in numerator and sum
    tol = (2.0 ** -8 + 2.0 ** -5) * mag + 2.0 ** -8 * want.abs()
    assert float((((got.double() - want).abs() - tol) / mag.amax()).max()) <= 0
