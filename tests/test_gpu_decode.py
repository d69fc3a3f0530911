"""GPU: the serving operators (include/dwa_decode.h) against plain formulas in
64 bits: the paged cache's write and read, attention of new tokens over it, and
the verification of drafted tokens.

Tolerance of the attention, per output: the probabilities are rounded to bf16
once (half a step, 2^-8 each) and so is the result (2^-8), the scores are f32
sums of d products (|ds| <= (d + 2) 2^-24 scale sum |q||k|, below 1e-4 for the
inputs here, in the numerator and in the sum: 2^-11 covers both), so
    |out - exact| <= (2^-8 + 2^-11) sum p |v| / sum p + 2^-8 |exact|.
(e4m3 caches: probabilities are rounded to 2^-12 and values to 2^-11 at most; keys rounded
to 2^-12 move a score by at most 2^-12 scale sum |q||k|, below 2^-9 here, in the numerator
and in the sum: together below 2^-8 + 2^-11 too.)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16


def _dev():
    return torch.device("cuda", 0)


def quantise(x):
    """e4m3 codes and f32 scales by the definition (f32 divisions)."""
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.clamp(amax / torch.full_like(amax, 448.0), min=2.0 ** -126)
    codes = (x / scale[..., None]).to(E4M3)
    bad = ~torch.isfinite(x).all(-1)
    scale[bad] = math.nan
    codes.view(torch.uint8)[bad] = 0
    return codes, scale


class Cache:
    """A filled cache; `dense(b)` gives sequence b's keys and values in 64 bits."""

    def __init__(self, kind, lengths, heads, d, page, seed, spare=3, poison=True):
        dev = _dev()
        g = torch.Generator(device=dev).manual_seed(seed)
        self.page, self.lengths = page, lengths
        used = [-(-n // page) for n in lengths]
        n_pages = sum(used) + spare
        shape = (n_pages, heads, page, d)
        self.k, self.v = (torch.randn(shape, device=dev, generator=g).to(BF16) for _ in range(2))
        self.k_scale = self.v_scale = None
        if kind == "e4m3":
            self.k, self.k_scale = quantise(self.k)
            self.v, self.v_scale = quantise(self.v * 3)
        order = torch.randperm(n_pages, device=dev, generator=g).int()
        self.table = torch.full((len(lengths), max(max(used), 1)), -7, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        if poison:  # what lies behind a sequence's end and in unused pages must not matter
            free = order[at:].long()
            bad = [self.k, self.v] if kind == "bf16" else [self.k_scale, self.v_scale]
            for x in bad:
                x[free] = math.nan
                for b, n in enumerate(lengths):
                    if n % page:
                        x[self.table[b, n // page].long(), :, n % page:] = math.nan
        self.len = torch.tensor(lengths, dtype=torch.int32, device=dev)

    def dense(self, b):
        n = self.lengths[b]
        ids = self.table[b, :-(-n // self.page)].long()
        out = []
        for x, s in ((self.k, self.k_scale), (self.v, self.v_scale)):
            y = x[ids].double()
            if s is not None:
                y = y * s[ids].double()[..., None]
            out.append(y.transpose(0, 1).flatten(1, 2)[:, :n])  # [H, n, d]
        return out

    def scales(self):
        return {} if self.k_scale is None else dict(k_scale=self.k_scale, v_scale=self.v_scale)


def attention_64(q, cache, start, scale=None):
    """(out, sum p |v| / sum p) in 64 bits for rows start[b]..start[b + 1]."""
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
        s = torch.einsum("nhd,hld->hnl", q[rows].double(), k) * scale
        see = torch.arange(length, device=q.device) < (length - n + 1 + torch.arange(n, device=q.device))[:, None]
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(see, torch.exp(s - top.clamp(min=-1e300)), 0.0)
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        out[rows] = torch.einsum("hnl,hld->nhd", p, v)
        mag[rows] = torch.einsum("hnl,hld->nhd", p, v.abs())
    return out, mag


def check(got, want, mag):
    assert not torch.isnan(got).any()
    tol = (2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -8 * want.abs()
    off = (got.double() - want).abs() - tol
    assert float(off.max()) <= 0, f"{float(off.max())} beyond the bound at {off.argmax().item()}"


def starts(new):
    return [sum(new[:b]) for b in range(len(new) + 1)]


def attend(cache, q, new, **kw):
    import computd_b200 as cb

    start = torch.tensor(starts(new), dtype=torch.int32, device=q.device)
    return cb.paged_attention(q, cache.k, cache.v, cache.table, cache.len, q_start=start,
                              max_q=max(max(new), 1), **cache.scales(), **kw)


# (new tokens, lengths): one token each; drafted tokens; an empty sequence, one without new
# tokens and one with more new tokens than cached ones; chunks that end inside a page
SHAPES = [
    ([1], [1]),
    ([1, 1, 1], [1, 17, 300]),
    ([1] * 5, [16, 33, 0, 128, 5]),
    ([3, 1, 5, 8], [3, 40, 129, 1000]),
    ([4, 0, 7, 2], [0, 9, 3, 50]),
    ([20, 33, 1], [20, 500, 64]),
    ([130, 257], [200, 257]),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 4, 64, 16), (2, 2, 128, 64), (8, 2, 128, 32),
                                                   (6, 1, 80, 16), (3, 3, 16, 128), (16, 1, 48, 64),
                                                   (5, 5, 112, 32)])
@pytest.mark.parametrize("new,lengths", SHAPES)
def test_paged_attention(kind, heads, kv_heads, d, page, new, lengths):
    dev = _dev()
    cache = Cache(kind, lengths, kv_heads, d, page, seed=len(new) + d)
    g = torch.Generator(device=dev).manual_seed(d + page)
    q = torch.randn((sum(new), heads, d), device=dev, generator=g).to(BF16)
    want, mag = attention_64(q, cache, starts(new))
    check(attend(cache, q, new), want, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,lengths", [([1, 1], [5000, 20001]), ([2, 6], [9000, 4097]),
                                         ([513], [6000])])
def test_paged_attention_long(kind, new, lengths):
    dev = _dev()
    cache = Cache(kind, lengths, 2, 128, 64, seed=9)
    g = torch.Generator(device=dev).manual_seed(3)
    q = (2 * torch.randn((sum(new), 8, 128), device=dev, generator=g)).to(BF16)
    want, mag = attention_64(q, cache, starts(new))
    check(attend(cache, q, new), want, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_paged_attention_layouts(kind, n):
    """q inside wider rows, out inside wider rows, rows behind the last sequence left alone,
    equal chunks without q_start, a scale of the caller's, pages of a shared tensor."""
    import computd_b200 as cb

    dev = _dev()
    lengths, H, d = [70, 200, 131], 4, 64
    cache = Cache(kind, lengths, 2, d, 32, seed=5)
    both = torch.stack([cache.k.view(torch.uint8), cache.v.view(torch.uint8)], 1)  # [pages, 2, H, page, bytes]
    cache.k, cache.v = (both[:, i].view(cache.k.dtype) for i in range(2))
    if kind == "e4m3":
        s = torch.stack([cache.k_scale, cache.v_scale], 1)
        cache.k_scale, cache.v_scale = s[:, 0], s[:, 1]
    g = torch.Generator(device=dev).manual_seed(1)
    wide = torch.randn((3 * n, 3 * H * d), device=dev, generator=g).to(BF16)
    q = wide[:, H * d:2 * H * d].view(3 * n, H, d)
    want, mag = attention_64(q, cache, [0, n, 2 * n, 3 * n], scale=0.3)
    out = torch.full((3 * n, 2 * H * d), 7.0, device=dev, dtype=BF16)
    dst = out[:, :H * d].view(3 * n, H, d)
    got = cb.paged_attention(q, cache.k, cache.v, cache.table, cache.len, scale=0.3, out=dst,
                             **cache.scales())
    assert got is dst
    check(got, want, mag)
    assert bool((out[:, H * d:] == 7).all())
    # only the first two sequences: the last n rows stay
    start = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev)
    out.fill_(5.0)
    cb.paged_attention(q, cache.k, cache.v, cache.table[:2], cache.len[:2], q_start=start, scale=0.3,
                       out=dst, **cache.scales())
    check(dst[:2 * n], want[:2 * n], mag[:2 * n])
    assert bool((dst[2 * n:] == 5).all())


@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_unseen_values_do_not_leak(n, d):
    """NaN and infinity in the last new token's key and value reach that token's rows and no other's."""
    dev = _dev()
    for kind in ("bf16", "e4m3"):
        lengths = [n + 11, n]
        cache = Cache(kind, lengths, 2, d, 16, seed=8)
        g = torch.Generator(device=dev).manual_seed(2)
        q = torch.randn((2 * n, 4, d), device=dev, generator=g).to(BF16)
        want, mag = attention_64(q, cache, [0, n, 2 * n])
        last = lengths[0] - 1
        page = cache.table[0, last // 16].long()
        if kind == "bf16":
            cache.v[page, 1, last % 16, 3] = math.inf
            cache.v[page, 1, last % 16, d - 1] = math.nan
        else:
            cache.v_scale[page, 1, last % 16] = math.nan
        got = attend(cache, q, [n, n])
        keep = torch.ones(2 * n, 4, d, dtype=torch.bool, device=dev)
        if kind == "bf16":
            for c in (3, d - 1):
                keep[n - 1, 2:, c] = False
        else:
            keep[n - 1, 2:] = False
        assert not bool(torch.isfinite(got[~keep]).any())
        check(torch.where(keep, got, 0).to(BF16), torch.where(keep, want, 0), mag)
        cache.k[page, 1, last % 16] = torch.full((d,), math.nan, device=dev).to(cache.k.dtype)
        if kind == "e4m3":
            cache.k_scale[page, 1, last % 16] = math.nan
        got = attend(cache, q, [n, n])
        keep[n - 1, 2:] = False
        assert not bool(torch.isfinite(got[~keep]).any())
        check(torch.where(keep, got, 0).to(BF16), torch.where(keep, want, 0), mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 3, 10])
@pytest.mark.parametrize("B,heads,d,longest", [(20, 4, 64, 256), (20, 4, 128, 512), (40, 8, 64, 300),
                                               (130, 2, 80, 200)])
def test_many_ragged_sequences(kind, n, B, heads, d, longest):
    """Every SM with one block, and with several that start longest first (or, for more sequences
    than are ranked, in their own order); lengths from nothing to `longest`."""
    dev = _dev()
    lengths = [(37 * b * b + 11 * b) % (longest + 1) for b in range(B - 1)] + [longest]
    cache = Cache(kind, lengths, heads, d, 32, seed=B + d)
    g = torch.Generator(device=dev).manual_seed(n)
    q = torch.randn((n * B, heads, d), device=dev, generator=g).to(BF16)
    want, mag = attention_64(q, cache, starts([n] * B))
    check(attend(cache, q, [n] * B), want, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,heads,d", [(4, 2, 128), (4, 2, 80), (7, 2, 48), (300, 1, 128), (300, 1, 64)])
def test_unseen_values_of_split_contexts(kind, n, heads, d):
    """The same where several blocks share the context: a value that is not finite in the middle of
    the new tokens."""
    dev = _dev()
    length = 7000
    cache = Cache(kind, [length], heads, d, 32, seed=d + n)
    g = torch.Generator(device=dev).manual_seed(n)
    q = torch.randn((n, 2 * heads, d), device=dev, generator=g).to(BF16)
    want, mag = attention_64(q, cache, [0, n])
    keep = torch.ones(n, 2 * heads, d, dtype=torch.bool, device=dev)
    at = length - n + n // 2
    page = cache.table[0, at // 32].long()
    if kind == "bf16":
        cache.v[page, 0, at % 32, 5] = -math.inf
        keep[n // 2:, :2, 5] = False
    else:
        cache.v_scale[page, 0, at % 32] = math.nan
        keep[n // 2:, :2] = False
    got = attend(cache, q, [n])
    assert not bool(torch.isfinite(got[~keep]).any())
    check(torch.where(keep, got, 0).to(BF16), torch.where(keep, want, 0), mag)


@pytest.mark.parametrize("n", [1, 5, 70])
def test_tiny_queries_and_large_keys(n):
    """Rows of q down to bf16's subnormal numbers against keys whose scales make up for it:
    the power of two that takes q into 16 bits loses nothing of them."""
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(n)
    cache = Cache("e4m3", [500, n], 2, 128, 64, seed=6, poison=False)
    cache.k_scale = cache.k_scale * 2.0 ** 120
    q = torch.randn((2 * n, 4, 128), device=dev, generator=g)
    q = (q * torch.exp2(torch.randint(-128, -122, (2 * n, 1, 1), device=dev, generator=g).float())).to(BF16)
    want, mag = attention_64(q, cache, [0, n, 2 * n], scale=1.0)
    check(attend(cache, q, [n, n], scale=1.0), want, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [16, 48, 80, 112])
@pytest.mark.parametrize("page", [16, 64])
def test_odd_rows_of_strided_pages(kind, d, page):
    """Rows of an odd number of 16 channels, in pages of a tensor that holds keys and values in turn."""
    dev = _dev()
    lengths, new = [1, 33, 700, 47], [1, 3, 2, 8]
    cache = Cache(kind, lengths, 3, d, page, seed=d)
    both = torch.stack([cache.k.view(torch.uint8), cache.v.view(torch.uint8)], 1)
    cache.k, cache.v = (both[:, i].view(cache.k.dtype) for i in range(2))
    g = torch.Generator(device=dev).manual_seed(page)
    q = torch.randn((sum(new), 3, d), device=dev, generator=g).to(BF16)
    want, mag = attention_64(q, cache, starts(new))
    check(attend(cache, q, new), want, mag)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 9, 140])
def test_sizes_far_apart(kind, n):
    """Values from 2^-24 to 2^24 and keys from 2^-16 to 1 from one token to the next, rows of q
    from 2^-100 to 2^20: 16-bit operands hold them relative to powers of two."""
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(n)
    cache = Cache(kind, [700, n + 3], 2, 128, 32, seed=21, poison=False)
    pages = cache.k.shape[0]
    kf = torch.exp2(torch.randint(-16, 1, (pages, 1, 32, 1), device=dev, generator=g).float())
    vf = torch.exp2(torch.randint(-24, 25, (pages, 1, 32, 1), device=dev, generator=g).float())
    if kind == "bf16":
        cache.k, cache.v = (cache.k.float() * kf).to(BF16), (cache.v.float() * vf).to(BF16)
    else:
        cache.k_scale, cache.v_scale = cache.k_scale * kf[..., 0], cache.v_scale * vf[..., 0]
    q = torch.randn((2 * n, 4, 128), device=dev, generator=g)
    q = (q * torch.exp2(torch.randint(-100, 1, (2 * n, 1, 1), device=dev, generator=g).float())).to(BF16)
    want, mag = attention_64(q, cache, [0, n, 2 * n])
    check(attend(cache, q, [n, n]), want, mag)
    # scores of 2^20 and more: one key takes all; ties of the products' roundings apart,
    # the outputs are that key's values
    big = (q.float().sign() * 2.0 ** 20).to(BF16)
    got = attend(cache, big, [n, n])
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 70])
def test_scale_zero_and_scores_of_minus_infinity(kind, n):
    dev = _dev()
    cache = Cache(kind, [n + 50, n], 2, 64, 16, seed=2)
    q = torch.randn((2 * n, 4, 64), device=dev).to(BF16)
    want, mag = attention_64(q, cache, [0, n, 2 * n], scale=0.0)
    check(attend(cache, q, [n, n], scale=0.0), want, mag)
    if kind == "bf16":  # every score is minus infinity: nothing is seen
        q, ids = torch.ones_like(q), cache.table[0, :cache.table.shape[1]].long()
        cache.k[ids] = -math.inf
        got = attend(cache, q, [n, n])
        assert bool((got[:n] == 0).all()) and bool(torch.isfinite(got[n:]).all())


def test_refused_arguments():
    """Wrong types, shapes, strides and devices raise before anything is launched."""
    import computd_b200 as cb

    dev = _dev()
    cache = Cache("e4m3", [40, 20], 2, 64, 16, seed=2)
    q = torch.zeros((2, 4, 64), device=dev, dtype=BF16)
    sc = cache.scales()
    good = dict(q=q, k_cache=cache.k, v_cache=cache.v, block_table=cache.table, lengths=cache.len)

    def attend_with(**kw):
        a = {**good, **sc, **kw}
        return cb.paged_attention(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("block_table"),
                                  a.pop("lengths"), **a)

    attend_with()
    bad = [dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q[0]), dict(q=q.transpose(0, 1)),
           dict(q=torch.zeros((3, 4, 64), device=dev, dtype=BF16)),  # not equal chunks
           dict(q=torch.zeros((2, 3, 64), device=dev, dtype=BF16)),  # 3 heads over 2
           dict(q=q.cpu()), dict(k_cache=cache.k.float()), dict(k_cache=cache.k[0]),
           dict(k_cache=cache.k.transpose(1, 2), v_cache=cache.v.transpose(1, 2)),
           dict(v_cache=cache.v[:1]), dict(k_scale=None), dict(v_scale=cache.v_scale.double()),
           dict(k_scale=cache.k_scale[:1]), dict(block_table=cache.table.long()),
           dict(block_table=cache.table[0]), dict(block_table=cache.table.cpu()),
           dict(lengths=cache.len.long()), dict(lengths=cache.len[:1]),
           dict(q_start=torch.zeros(2, dtype=torch.int32, device=dev)),
           dict(max_q=0), dict(scale=-1.0), dict(scale=math.nan), dict(out=q.float()),
           dict(out=torch.zeros((2, 4, 128), device=dev, dtype=BF16)[:, :, ::2]),
           dict(status=torch.zeros(2, dtype=torch.int32, device=dev)),
           dict(q=q.clone().requires_grad_())]
    for kw in bad:
        with pytest.raises(ValueError):
            attend_with(**kw)
    with pytest.raises(TypeError):
        attend_with(q=[1])
    k = torch.zeros((5, 2, 64), device=dev, dtype=BF16)
    slots = torch.arange(5, device=dev)
    for a in [(k.half(), k.half()), (k, k.float()), (k[:, :1], k[:, :1]), (k, k[:4]),
              (k[:, :, ::2], k[:, :, ::2]), (k.cpu(), k.cpu())]:
        with pytest.raises(ValueError):
            cb.kv_cache_write(*a, cache.k, cache.v, slots, **sc)
    for s in (slots.int(), slots[:4], slots[None], torch.arange(10, device=dev)[::2]):
        with pytest.raises(ValueError):
            cb.kv_cache_write(k, k, cache.k, cache.v, s, **sc)
    with pytest.raises(ValueError):  # rows that do not start on 16 bytes
        wide = torch.zeros((5, 2, 65), device=dev, dtype=BF16)
        cb.kv_cache_write(wide[:, :, 1:], wide[:, :, 1:], cache.k, cache.v, slots, **sc)
    with pytest.raises(ValueError):
        cb.kv_cache_read(cache.k, cache.v, slots, out=(k.float(), k), **sc)
    odd = torch.zeros((4, 2, 16, 24), device=dev, dtype=BF16)
    with pytest.raises(cb.DWAArgumentError):
        cb.kv_cache_read(odd, odd, slots)
    p = torch.zeros((2, 3, 9), device=dev)
    x, u, r = torch.zeros((2, 2), dtype=torch.int32, device=dev), p[:, :2, 0].contiguous(), p[:, 0, 0].contiguous()
    cb.verify_drafts(p, x, p[:, :2].contiguous(), u, r)
    for a in [(p.half(), x, None, u, r), (p, x.long(), None, u, r), (p, x, p[:, :2], u, r),
              (p, x, p[:, :2].bfloat16(), u, r), (p, x, None, u[:1], r), (p, x, None, u, u),
              (p.cpu(), x, None, u, r), (p[:, :, ::2], x, None, u, r)]:
        with pytest.raises(ValueError):
            cb.verify_drafts(*a)


@pytest.mark.parametrize("n", [1, 6, 150])
def test_bad_tables_and_lengths(n):
    """Bad page numbers, lengths and row ranges: NaN rows for their sequence alone, and the status."""
    import computd_b200 as cb

    dev = _dev()
    lengths = [150 + n] * 4
    cache = Cache("bf16", lengths, 2, 64, 16, seed=4)
    q = torch.randn((4 * n, 4, 64), device=dev).to(BF16)
    want, mag = attention_64(q, cache, starts([n] * 4))
    start = torch.tensor(starts([n] * 4), dtype=torch.int32, device=dev)

    def run(table, length, q_start, bad, max_q=n):
        status = torch.zeros((), dtype=torch.int32, device=dev)
        out = torch.full((4 * n, 4, 64), 3.0, device=dev, dtype=BF16)
        cb.paged_attention(q, cache.k, cache.v, table, length, q_start=q_start, max_q=max_q, out=out,
                           status=status)
        assert status.item() == (5 if bad else 0)
        for b in range(4):
            rows = slice(b * n, (b + 1) * n)
            if b in bad:
                assert bool(torch.isnan(out[rows]).all())
            else:
                check(out[rows], want[rows], mag[rows])
        return out

    run(cache.table, cache.len, start, [])
    for page in (-1, cache.k.shape[0], 2 ** 31 - 1):
        table = cache.table.clone()
        table[2, 1] = page
        run(table, cache.len, start, [2])
    for length in (-1, cache.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        lens = cache.len.clone()
        lens[1] = length
        run(cache.table, lens, start, [1])
    if n > 1:
        run(cache.table, cache.len, start, [0, 1, 2, 3], max_q=n - 1)
    # a row range outside q: nothing of that sequence is written
    status = torch.zeros((), dtype=torch.int32, device=dev)
    out = torch.full((4 * n, 4, 64), 3.0, device=dev, dtype=BF16)
    bad = start.clone()
    bad[4] = 4 * n + 1
    cb.paged_attention(q, cache.k, cache.v, cache.table, cache.len, q_start=bad, max_q=n, out=out,
                       status=status)
    assert status.item() == 5
    check(out[:3 * n], want[:3 * n], mag[:3 * n])
    assert bool((out[3 * n:] == 3).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("src", [BF16, torch.float32])
@pytest.mark.parametrize("T,heads,d,page", [(1, 1, 16, 16), (7, 3, 80, 16), (300, 16, 64, 32),
                                            (2000, 4, 128, 128), (65, 5, 48, 64)])
def test_write_and_read(kind, src, T, heads, d, page):
    import computd_b200 as cb

    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(T + d)
    n_pages = -(-T // page) + 3
    x = torch.randn((T, 3 * heads * d), device=dev, generator=g).mul_(
        torch.logspace(-20, 20, T, device=dev)[:, None]).to(src)
    k = x[:, heads * d:2 * heads * d].view(T, heads, d)
    v = x[:, 2 * heads * d:].view(T, heads, d).transpose(0, 1).contiguous().transpose(0, 1)
    k[0] = 0
    if T > 5:
        k[2, 0, 1], k[3, -1, d - 1], v[4, 0, 0] = math.nan, math.inf, -math.inf
        v[5, 0] = 2.0 ** -130  # below the smallest scale
    slots = torch.randperm(n_pages * page, device=dev, generator=g)[:T]
    shape = (n_pages, heads, page, d)
    dtype = E4M3 if kind == "e4m3" else BF16
    kc, vc = (torch.full(shape, 2.0, device=dev).to(dtype) for _ in range(2))
    sc = [torch.full(shape[:3], 9.0, device=dev) if kind == "e4m3" else None for _ in range(2)]
    status = torch.zeros((), dtype=torch.int32, device=dev)
    want = []
    for y, c, s in ((k, kc, sc[0]), (v, vc, sc[1])):
        c, s = c.clone(), None if s is None else s.clone()
        at, off = slots // page, slots % page
        if kind == "e4m3":
            codes, scales = quantise(y)
            c.view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            s[at, :, off] = scales
        else:
            c[at, :, off] = y.to(BF16)
        want.append((c, s))
    cb.kv_cache_write(k, v, kc, vc, slots, k_scale=sc[0], v_scale=sc[1], status=status)
    assert status.item() == 0
    for (c, s), got, gs in zip(want, (kc, vc), sc):
        bits = torch.uint8 if kind == "e4m3" else torch.int16
        if kind == "bf16":  # any NaN will do
            got, c = torch.where(torch.isnan(got), 1.0, got), torch.where(torch.isnan(c), 1.0, c)
        assert torch.equal(got.view(bits), c.view(bits))
        if s is not None:
            assert torch.equal(torch.nan_to_num(gs, nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    back = cb.kv_cache_read(kc, vc, slots, k_scale=sc[0], v_scale=sc[1], status=status)
    assert status.item() == 0
    for got, y, c, s in zip(back, (k, v), (kc, vc), sc):
        at, off = slots // page, slots % page
        if kind == "bf16":
            torch.testing.assert_close(got, y.to(BF16), rtol=0, atol=0, equal_nan=True)
        else:
            codes = c.view(torch.uint8)[at, :, off].view(E4M3).float()
            torch.testing.assert_close(got, (codes * s[at, :, off][..., None]).to(BF16), rtol=0,
                                       atol=0, equal_nan=True)
            # half a step of e4m3 (2^-4, or 2^-10 of the scale near zero), then of bf16
            fine = torch.isfinite(y).all(-1)
            off_by = (got.double() - y.double()).abs()[fine]
            bound = (2.0 ** -4 + 2.0 ** -8) * y.double().abs() + 2.0 ** -10 * s[at, :, off][..., None].double()
            assert bool((off_by <= 1.01 * bound[fine]).all())
            assert bool(torch.isnan(got[~fine]).all())


def test_write_repeated_skipped_and_bad_slots():
    import computd_b200 as cb

    dev = _dev()
    for T in (6, 500, 9000):
        g = torch.Generator(device=dev).manual_seed(T)
        heads, d, page, n_pages = 2, 32, 16, 8
        n = n_pages * page
        k, v = (torch.randn((T, heads, d), device=dev, generator=g).to(BF16) for _ in range(2))
        slots = torch.randint(-1, n, (T,), device=dev, generator=g)
        slots[1], slots[3] = n, -2
        kc = torch.zeros((n_pages, heads, page, d), device=dev, dtype=BF16)
        vc = torch.zeros_like(kc)
        want_k, want_v = kc.clone(), vc.clone()
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < n:
                want_k[s // page, :, s % page], want_v[s // page, :, s % page] = k[t], v[t]
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        cb.kv_cache_write(k, v, kc, vc, slots, status=status)
        assert status.item() == 5
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
        # read: skipped rows zero, or left as they were; bad ones NaN
        status.zero_()
        got, _ = cb.kv_cache_read(kc, vc, slots, status=status)
        assert status.item() == 5
        fine = (slots >= 0) & (slots < n)
        at, off = slots.clamp(0, n - 1) // page, slots.clamp(0, n - 1) % page
        assert torch.equal(got[fine], kc[at, :, off][fine])
        assert bool((got[slots == -1] == 0).all())
        assert bool(torch.isnan(got[[1, 3]]).all())
        out = tuple(torch.full((T, heads, d), 4.0, device=dev, dtype=BF16) for _ in range(2))
        cb.kv_cache_read(kc, vc, slots, out=out)
        assert bool((out[1][slots == -1] == 4).all())
        assert torch.equal(out[1][fine], vc[at, :, off][fine])


def test_cache_beyond_32_bit_offsets():
    """A cache of 5 GB for keys and as much for values: the last pages are written, read, attended to."""
    import computd_b200 as cb

    dev = _dev()
    heads, page, d = 8, 64, 128
    n_pages = 5 * 2 ** 30 // (heads * page * d)
    kc, vc = (torch.zeros((n_pages, heads, page, d), device=dev, dtype=E4M3) for _ in range(2))
    ks, vs = (torch.zeros((n_pages, heads, page), device=dev) for _ in range(2))
    T = 200
    g = torch.Generator(device=dev).manual_seed(0)
    k, v = (torch.randn((T, heads, d), device=dev, generator=g).to(BF16) for _ in range(2))
    pages = torch.tensor([n_pages - 1, n_pages // 2 + 5, 3, n_pages - 2], dtype=torch.int32, device=dev)
    t = torch.arange(T, device=dev)
    slots = pages.long()[t // page] * page + t % page
    cb.kv_cache_write(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
    rk, rv = cb.kv_cache_read(kc, vc, slots, k_scale=ks, v_scale=vs)
    for got, x in ((rk, k), (rv, v)):
        codes, scale = quantise(x)
        torch.testing.assert_close(got, (codes.float() * scale[..., None]).to(BF16), rtol=0, atol=0)
    for n in (1, 70):
        q = torch.randn((n, heads, d), device=dev, generator=g).to(BF16)
        cache = Cache.__new__(Cache)
        cache.k, cache.v, cache.k_scale, cache.v_scale = kc, vc, ks, vs
        cache.table, cache.page, cache.lengths = pages[None], page, [T]
        cache.len = torch.tensor([T], dtype=torch.int32, device=dev)
        want, mag = attention_64(q, cache, [0, n])
        check(attend(cache, q, [n]), want, mag)


@pytest.mark.parametrize("n", [1, 90])
def test_graphs_and_streams(n):
    """Captured calls follow their inputs; two graphs replayed on two streams at once do not meet."""
    import computd_b200 as cb

    dev = _dev()
    sets = []
    for seed in (1, 2):
        cache = Cache("e4m3", [700, 130], 4, 128, 32, seed=seed)
        q = torch.randn((2 * n, 16, 128), device=dev).to(BF16)
        start = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev)
        call = lambda q=q, c=cache, s=start: cb.paged_attention(  # noqa: E731
            q, c.k, c.v, c.table, c.len, q_start=s, max_q=n, **c.scales())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = call()
        torch.cuda.current_stream().wait_stream(side)
        sets.append((cache, q, side, graph, out, eager, start))
    torch.cuda.synchronize()
    for _ in range(20):
        for _, _, side, graph, _, _, _ in sets:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for cache, q, side, graph, out, eager, _ in sets:
        assert torch.equal(out, eager)
        want, mag = attention_64(q, cache, [0, n, 2 * n])
        check(out, want, mag)
        cache.len.copy_(torch.tensor([650, 91], dtype=torch.int32))
        cache.lengths = [650, 91]
        graph.replay()
        want, mag = attention_64(q, cache, [0, n, 2 * n])
        torch.cuda.synchronize()
        check(out, want, mag)


def verify_64(p, q, x, u, r, lengths):
    B, K1, V = p.shape
    kept_all, rows = [], []
    ok = lambda t: torch.where((t > 0) & torch.isfinite(t), t, 0.0)  # noqa: E731
    for b in range(B):
        n = min(max(int(lengths[b]), 0), K1 - 1)
        pb = ok(p[b].double())
        qb = ok(q[b].double()) if q is not None else None
        row, w = [], None
        for i in range(n):
            t = int(x[b, i])
            inside = 0 <= t < V
            one = torch.zeros(V, dtype=torch.float64)
            if inside:
                one[t] = 1
            qi = qb[i] if qb is not None else one
            if not (inside and float(u[b, i]) * float(qi[t]) < float(pb[i, t])):
                w = (pb[i] - qi).clamp(min=0)
                break
            row.append(t)
        if w is None or float(w.sum()) == 0:
            w = pb[len(row)]
        c = w.cumsum(0)
        kept_all.append(len(row))
        if float(c[-1]) == 0:
            row.append(-1)
        else:
            past = (c > float(r[b]) * float(c[-1])).nonzero()
            row.append(int(past[0]) if len(past) else int((w > 0).nonzero()[-1]))
        rows.append(row + [-1] * (K1 - len(row)))
    return kept_all, rows


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_outputs_of_their_own(mode):
    """A call's outputs are contiguous, overlap nothing, and are ordinary tensors of the mode."""
    import computd_b200 as cb

    dev = _dev()
    cache = Cache("bf16", [40], 3, 16, 16, seed=2)
    slots = torch.arange(7, device=dev)

    def same(x, y):  # bit for bit: page 0 is not in use and holds NaN
        return torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))

    probs = torch.full((5, 3, 9), 1 / 9, device=dev)
    with mode():
        k, v = cb.kv_cache_read(cache.k, cache.v, slots)
        n, tokens = cb.verify_drafts(probs, torch.zeros((5, 2), dtype=torch.int32, device=dev), None,
                                     torch.zeros((5, 2), device=dev), torch.zeros(5, device=dev))
        o = attend(cache, torch.zeros((1, 3, 16), device=dev, dtype=BF16), [1])
        for x, y in ((k, v), (tokens, n)):
            assert x.is_contiguous() and y.is_contiguous() and x.is_inference() == torch.is_inference_mode_enabled()
            assert y.data_ptr() >= x.data_ptr() + x.numel() * x.element_size()
            kept = y.clone()
            x.fill_(1)
            x.record_stream(torch.cuda.Stream())
            assert same(y, kept)
        assert o.shape == (1, 3, 16) and o.is_contiguous() and not o.requires_grad
        assert k.shape == v.shape == (7, 3, 16) and n.shape == (5,) and tokens.shape == (5, 3)
        assert same(v, cache.v[0].transpose(0, 1)[:7])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (9, 1, 65), (5, 0, 1), (40, 7, 2001), (3, 40, 64400),
                                   (300, 3, 130)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_drafts(dtype, B, K, V, certain):
    import computd_b200 as cb

    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(V + B)
    logits = 2 * torch.randn((B, K + 1, V), device=dev, generator=g)
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :K] + 0.3 * torch.randn((B, K, V), device=dev, generator=g), -1)
    x = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, K).int() if K else \
        torch.zeros((B, 0), dtype=torch.int32, device=dev)
    if certain:  # the drafter's best token; the target likes it
        p[:, :K] = 0.3 * p[:, :K] + 0.7 * torch.nn.functional.one_hot(x.long(), V)
    p, q = p.to(dtype), q.to(dtype)
    u = torch.rand((B, K), device=dev, generator=g)
    r = torch.rand((B,), device=dev, generator=g)
    lengths = torch.randint(-1, K + 2, (B,), device=dev, generator=g).int()
    if B > 4:
        r[0] = 0.0
        r[1] = 1 - 2.0 ** -24
        lengths[:4] = K
        if K:
            u[1, 0] = 1 - 2.0 ** -24
            x[2, 0] = V           # outside the vocabulary: falls
            p[3, :] = q[3, :1]    # p = q: nothing is left of p - q where a draft falls
            x[3, 0] = -3
            p[4, :] = 0           # no mass at all
            if V > 4:
                p[0, 0, :3] = torch.tensor([math.nan, math.inf, -1.0], device=dev)
    args = (x, None if certain else q, u, r)
    kept, tokens = cb.verify_drafts(p, *args, draft_lengths=lengths)
    again = cb.verify_drafts(p, *args, draft_lengths=lengths)
    want_kept, want = verify_64(p.cpu(), None if certain else q.cpu(), x.cpu(), u.cpu(), r.cpu(),
                                lengths.cpu())
    assert kept.tolist() == want_kept
    assert tokens.tolist() == want
    assert torch.equal(kept, again[0]) and torch.equal(tokens, again[1])
    full, _ = cb.verify_drafts(p, *args)
    assert bool((full >= kept).all())


def test_verified_tokens_follow_the_target():
    """Drafts from q, verified with fresh numbers: the first token of 60000 rounds is distributed as
    the target's p (each count within 5 of its standard deviations)."""
    import computd_b200 as cb

    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(11)
    B, V = 60000, 12
    p1 = torch.softmax(1.5 * torch.randn(V, device=dev, generator=g), -1)
    q1 = torch.softmax(1.5 * torch.randn(V, device=dev, generator=g), -1)
    p = p1.expand(B, 2, V).contiguous()
    q = q1.expand(B, 1, V).contiguous()
    x = torch.multinomial(q1, B, replacement=True, generator=g).int()[:, None]
    u, r = torch.rand((B, 1), device=dev, generator=g), torch.rand((B,), device=dev, generator=g)
    _, tokens = cb.verify_drafts(p, x, q, u, r)
    counts = torch.bincount(tokens[:, 0].long(), minlength=V).double()
    sd = torch.sqrt(B * p1.double() * (1 - p1.double()))
    assert bool(((counts - B * p1.double()).abs() <= 5 * sd).all())
