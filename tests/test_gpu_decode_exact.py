"""GPU: what the few-rows attention rounds, and that the chunk forward is the whole forward.

Over a bf16 cache the few-rows attention uses each probability as the sum of two bf16
numbers, 2^-17 of it off at most; the scores' f32 sums move it by at most 2^-13 for the inputs
here (d 2^-24 scale sum |q||k| in the numerator and in the sum, below 130 * 8 * 2^-24), so

    |out - exact| <= 2^-12 sum p |v| / sum p + 2^-8 |exact|,

the last the result's own rounding.  With one bf16 number the first term would be 2^-8.
"""
import pytest
import torch

from test_gpu_decode import BF16, Cache, attend, attention_64, starts

pytestmark = pytest.mark.gpu


def _once_rounded(q, cache, start):
    """The formula in 64 bits, but for probabilities (relative to the largest) rounded to bf16."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(cache.lengths):
        n = start[b + 1] - start[b]
        k, v = cache.dense(b)
        k, v = (x.repeat_interleave(q.shape[1] // k.shape[0], 0) for x in (k, v))
        s = torch.einsum("nhd,hld->hnl", q[start[b]:start[b + 1]].double(), k) * q.shape[2] ** -0.5
        see = torch.arange(length, device=q.device) < (length - n + 1 + torch.arange(n, device=q.device))[:, None]
        s = s.masked_fill(~see, -torch.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[start[b]:start[b + 1]] = torch.einsum("hnl,hld->nhd", p.to(BF16).double(), v) / \
            p.sum(-1).transpose(0, 1)[..., None]
    return out


@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 3, 80, 16), (4, 4, 128, 64)])
@pytest.mark.parametrize("new,lengths", [([1] * 6, [2, 3, 5, 9, 17, 33]), ([2, 3, 4], [3, 40, 12]),
                                         ([1, 2], [700, 3000])])
def test_few_rows_keep_their_probabilities(heads, kv_heads, d, page, new, lengths):
    cache = Cache("bf16", lengths, kv_heads, d, page, seed=d + len(new))
    g = torch.Generator("cuda").manual_seed(page)
    q = torch.randn((sum(new), heads, d), device="cuda", generator=g).to(BF16)
    want, mag = attention_64(q, cache, starts(new))
    bound = 2.0 ** -12 * mag + 2.0 ** -8 * want.abs()
    got = attend(cache, q, new)
    assert bool(((got.double() - want).abs() <= bound).all())
    if max(lengths) < 100:  # the bound tells the two apart
        assert bool(((_once_rounded(q, cache, starts(new)).to(BF16).double() - want).abs() > bound).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("r,dh", [(0, 32), (0, 80), (2, 16)])
def test_extend_is_the_forward_with_its_attention(monkeypatch, r, dh, dtype):
    """Whole sequences in one chunk: with every block's attention output put in the place of the whole
    forward's own, that one's logits are the chunk's bit for bit.  (The attention itself is held
    against 64 bits elsewhere.)"""
    from test_gpu_lm_extend import Recorder, _i32, _model, _table, _tokens

    cfg, model = _model(r, dh)
    tokens, cache = _tokens(cfg), model.new_cache(24, page_size=16, dtype=dtype)
    rec = Recorder(model)
    got = model.extend(tokens.reshape(-1), cache, _table(cfg, cache), _i32([cfg.seq_len] * cfg.batch))
    rec.close()
    layer = iter(range(cfg.n_layers))
    asked = []

    def recorded(q, k, v, is_causal):
        assert is_causal
        asked.append((q, k, v))
        return rec.o[next(layer)].view(cfg.batch, cfg.seq_len, cfg.n_heads, dh).transpose(1, 2)

    monkeypatch.setattr(torch.nn.functional, "scaled_dot_product_attention", recorded)
    whole = model(tokens)
    assert torch.equal(whole.view(-1, cfg.vocab), got)
    if dtype is torch.bfloat16:  # and its keys and values are what the cache holds
        slots, _ = cache.slots(_table(cfg, cache), _i32([cfg.seq_len] * cfg.batch),
                               _i32([cfg.seq_len * b for b in range(cfg.batch + 1)]), cfg.tokens)
        for i, (_, k, v) in enumerate(asked):
            ck, cv = cache.read(i, slots)
            assert torch.equal(k.transpose(1, 2).reshape(ck.shape), ck)
            assert torch.equal(v.transpose(1, 2).reshape(cv.shape), cv)
