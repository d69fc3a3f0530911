"""GPU: the language model over the paged cache (``DWALM.extend``, ``DWALM.verify``): the
cache's write, the attention that reads it and the draft verification run together.

Every block of a call is checked on its own input: the cache must hold exactly the
keys (rotated to their positions) and values of the tokens, or exactly their e4m3
codes and scales, and the attention's output must be the 64-bit formula's over the
cached tokens within its roundings (the bf16 probabilities' and the result's half
steps 2^-8, 2^-11 for f32, as in test_gpu_decode.py).  What follows in a block is the
code of the whole forward.  ``verify`` must decide as the 64-bit rule does on the
probabilities of the same (deterministic) ``extend``.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(r=0, dh=32, layers=2, seed=3):
    import computd_b200 as cb
    from computd_b200.dwa_lm import DWALM, DWALMConfig

    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    cfg = DWALMConfig(vocab=65, d_model=4 * dh, n_layers=layers, n_heads=4, seq_len=64, batch=3,
                      pool_rows=512, top_k=8, S=2, d_k=2 * dh, r=r)
    if r:
        return cfg, DWALM(cfg, None, cb.new_normal(cfg.pool_rows, cfg.D, seed=seed, stddev=0.3, device=dev))
    keys = cb.new_normal(cfg.pool_rows, cfg.key_width, seed=seed, stddev=cfg.key_width ** -0.5, device=dev)
    values = cb.new_normal(cfg.pool_rows, cfg.d_model, seed=seed + 1, stddev=cfg.d_model ** -0.5, device=dev)
    return cfg, DWALM(cfg, keys, values)


def _tokens(cfg, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, cfg.vocab, (cfg.batch, cfg.seq_len), device="cuda", generator=g)


def _table(cfg, cache, seed=1):
    pages = -(-cfg.seq_len // cache.page_size) + 1
    order = torch.randperm(cache.n_pages, generator=torch.Generator().manual_seed(seed))
    return order[:cfg.batch * pages].view(cfg.batch, pages).int().cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Recorder:
    """The attention inputs and outputs of every block in a call."""

    def __init__(self, model):
        self.model, self.x, self.o = model, {}, {}
        self.hooks = []
        for i, blk in enumerate(model.blocks):
            keep = lambda to, i: lambda m, inp: to.__setitem__(i, inp[0].detach().clone())  # noqa: E731
            self.hooks += [blk.attn.norm.register_forward_pre_hook(keep(self.x, i)),
                           blk.attn.proj.register_forward_pre_hook(keep(self.o, i))]

    def close(self):
        for h in self.hooks:
            h.remove()

    def check(self, cache, table, lengths, new):
        """Rows b's tokens lengths[b] - new[b] .. lengths[b] - 1, packed."""
        from test_gpu_decode import attention_64, check, quantise

        from computd_b200.lm_ops import rope_qk

        start = [sum(new[:b]) for b in range(len(new) + 1)]
        positions = torch.tensor([lengths[b] - new[b] + i for b in range(len(new)) for i in range(new[b])],
                                 device="cuda")
        page = cache.page_size
        slots = torch.cat([table[b, p // page].long() * page + p % page
                           for b in range(len(new))
                           for p in [positions[start[b]:start[b + 1]]]])
        n = start[-1]
        for i, blk in enumerate(self.model.blocks):
            attn = blk.attn
            x, o = self.x[i], self.o[i]
            T, C = x.shape[1:]
            qkv = attn.qkv(attn.norm(x))
            cos, sin = (t[torch.cat([positions, positions.new_zeros(T - n)])] for t in (attn.cos, attn.sin))
            q, k = (t.transpose(1, 2)[0, :n] for t in rope_qk(qkv, cos, sin, attn.h, attn.dh))
            v = qkv[0, :n, 2 * C:].view(n, attn.h, attn.dh)
            at, off = slots // page, slots % page
            for y, held, scale in ((k, cache.k[i], cache.k_scale), (v, cache.v[i], cache.v_scale)):
                if scale is None:
                    assert torch.equal(held[at, :, off], y)
                else:
                    codes, scales = quantise(y)
                    assert torch.equal(held.view(torch.uint8)[at, :, off], codes.view(torch.uint8))
                    assert torch.equal(scale[i][at, :, off], scales)

            class Dense:
                pass

            dense = Dense()
            dense.lengths = lengths

            def of(b, i=i):
                ids = table[b, :-(-lengths[b] // page)].long()
                out = []
                for held, scale in ((cache.k[i], cache.k_scale), (cache.v[i], cache.v_scale)):
                    y = held[ids].double()
                    if scale is not None:
                        y = y * scale[i][ids].double()[..., None]
                    out.append(y.transpose(0, 1).flatten(1, 2)[:, :lengths[b]])
                return out

            dense.dense = of
            want, mag = attention_64(q, dense, start)
            check(o[0, :n].view(n, attn.h, attn.dh), want, mag)


@pytest.mark.parametrize("r,dh", [(0, 32), (0, 80), (2, 16)])
@pytest.mark.parametrize("chunks", [[64], [1] * 64, [40, 1, 1, 7, 15], [16, 48]])
def test_extend_block_by_block(r, dh, chunks):
    cfg, model = _model(r, dh)
    tokens = _tokens(cfg)
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    rec = Recorder(model)
    at = 0
    for n in chunks:
        at += n
        out = model.extend(tokens[:, at - n:at].reshape(-1), cache, table, _i32([at] * cfg.batch))
        assert out.shape == (cfg.batch * n, cfg.vocab) and bool(torch.isfinite(out).all())
        rec.check(cache, table, [at] * cfg.batch, [n] * cfg.batch)
    rec.close()
    cache.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_uneven_chunks_and_padding(dtype):
    """Sequences at different places in one call, rows behind the last one, both cache types."""
    cfg, model = _model()
    tokens = _tokens(cfg, 5)
    cache = model.new_cache(24, page_size=32, dtype=dtype)
    table = _table(cfg, cache)
    rec = Recorder(model)
    length = [0, 0, 0]
    for new in ([30, 1, 64], [0, 40, 0], [34, 23, 0]):
        rows = [tokens[b, length[b]:length[b] + n] for b, n in enumerate(new)]
        pad = torch.zeros(100 - sum(new), dtype=torch.long, device="cuda")
        length = [a + n for a, n in zip(length, new)]
        start = [sum(new[:b]) for b in range(4)]
        out = model.extend(torch.cat(rows + [pad]), cache, table, _i32(length), _i32(start), max(new))
        assert bool(torch.isfinite(out[:start[-1]]).all())
        rec.check(cache, table, length, new)
    rec.close()
    assert length == [64, 64, 64]
    cache.check()


def test_one_token_of_one_sequence():
    cfg, model = _model()
    cache = model.new_cache(4, page_size=16)
    table = _i32([[2, 0, 1]])
    rec = Recorder(model)
    for n in range(1, 20):
        out = model.extend(_tokens(cfg)[0, n - 1:n], cache, table, _i32([n]))
        assert out.shape == (1, cfg.vocab)
        rec.check(cache, table, [n], [1])
    rec.close()
    assert model.extend(_tokens(cfg)[0, :0], cache, table, _i32([5]), _i32([0, 0])).shape == (0, cfg.vocab)
    with pytest.raises(ValueError):
        model.extend(_tokens(cfg)[0, :3], cache, _table(cfg, model.new_cache(24, page_size=16)), _i32([3, 1]))
    cache.check()


def test_extend_in_a_graph():
    cfg, model = _model(layers=3)
    tokens = _tokens(cfg, 7)
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    model.extend(tokens[:, :40].reshape(-1), cache, table, _i32([40] * 3))
    ids, lengths = tokens[:, 40].clone(), _i32([41] * 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            model.extend(ids, cache, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.extend(ids, cache, table, lengths)
    for at in range(41, 46):
        ids.copy_(tokens[:, at])
        lengths.fill_(at + 1)
        graph.replay()
        got = out.clone()
        eager = model.extend(ids, cache, table, lengths)
        assert torch.equal(got, eager)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_decides_on_the_models_probabilities(dtype, certain):
    """Drafts scored in one chunk: the outcome is the 64-bit rule's on that chunk's softmax, the
    lengths returned are what stays, and the next token is attended from there."""
    from test_gpu_decode import verify_64

    cfg, model = _model(seed=9)
    tokens = _tokens(cfg, 11)
    n0, K, B, V = [20, 33, 7], 4, cfg.batch, cfg.vocab
    cache = model.new_cache(24, page_size=16, dtype=dtype)
    table = _table(cfg, cache)
    rows = torch.cat([tokens[b, :n] for b, n in enumerate(n0)])
    start = _i32([0, 20, 53, 60])
    model.extend(rows, cache, table, _i32(n0), start, max(n0))
    g = torch.Generator(device="cuda").manual_seed(1)
    last = torch.stack([tokens[b, n] for b, n in enumerate(n0)])
    lengths = _i32(n0)
    for step in range(3):
        q = torch.softmax(torch.randn((B, K, V), device="cuda", generator=g), -1)
        drafts = torch.multinomial(q.view(B * K, V), 1, generator=g).view(B, K).int()
        u = torch.rand((B, K), device="cuda", generator=g) * (0.05 if step else 1.0)
        r = torch.rand((B,), device="cuda", generator=g)
        chunk = torch.cat([last.view(B, 1), drafts.long()], 1).reshape(-1)
        logits = model.extend(chunk, cache, table, lengths + (K + 1))
        probs = torch.softmax(logits.float().view(B, K + 1, -1) / 0.7, -1)
        accepted, out, new = model.verify(last, drafts, None if certain else q, u, r, cache, table, lengths,
                                          temperature=0.7)
        kept, want = verify_64(probs.cpu(), None if certain else q.cpu(), drafts.cpu(), u.cpu(), r.cpu(),
                               [K] * B)
        assert accepted.tolist() == kept and out.tolist() == want
        assert new.tolist() == [a + 1 + k for a, k in zip(lengths.tolist(), kept)]
        last = torch.stack([out[b, kept[b]] for b in range(B)]).long()
        lengths = new
    rec = Recorder(model)
    model.extend(last, cache, table, lengths + 1)
    rec.check(cache, table, (lengths + 1).tolist(), [1] * B)
    rec.close()
    cache.check()


@pytest.mark.parametrize("certain", [False, True])
def test_drafts_outside_the_vocabulary_fall(certain):
    """What follows a sequence's drafts, and drafts outside the vocabulary, reach no table; the
    outcome is the 64-bit rule's on the model's probabilities."""
    from test_gpu_decode import verify_64

    cfg, model = _model(seed=4)
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    tokens = _tokens(cfg, 2)
    model.extend(tokens[:, :9].reshape(-1), cache, table, _i32([9] * 3))
    drafts = _i32([[5, 7, -1], [-1, -1, -1], [3, cfg.vocab, 2]])
    u, r = torch.zeros((3, 3), device="cuda"), torch.full((3,), 0.5, device="cuda")
    q = None if certain else torch.full((3, 3, cfg.vocab), 1 / 64, device="cuda")
    last = tokens[:, 9]
    chunk = torch.cat([last.view(3, 1), drafts.clamp(0, cfg.vocab - 1).long()], 1).reshape(-1)
    logits = model.extend(chunk, cache, table, _i32([13] * 3))
    probs = torch.softmax(logits.float().view(3, 4, -1), -1)
    accepted, out, new = model.verify(last, drafts, q, u, r, cache, table, _i32([9] * 3),
                                      draft_lengths=_i32([2, 0, 3]))
    kept, want = verify_64(probs.cpu(), None if certain else q.cpu(), drafts.cpu(), u.cpu(), r.cpu(), [2, 0, 3])
    assert kept == [2, 0, 1]
    assert accepted.tolist() == kept and out.tolist() == want and new.tolist() == [12, 10, 11]


@pytest.mark.parametrize("max_q", [2, 40])
def test_padding_rows_attend_to_nothing(max_q):
    """Whatever the allocator hands out: the rows behind the last sequence are finite."""
    cfg, model = _model()
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    tokens = _tokens(cfg)[:, :2].reshape(-1)
    pad = torch.zeros(34, dtype=torch.long, device="cuda")
    start = _i32([0, 2, 4, 6])
    rec = Recorder(model)
    for _ in range(3):
        junk = [torch.full((40, cfg.d_model), float("nan"), dtype=torch.bfloat16, device="cuda")
                for _ in range(20)]
        del junk
        out = model.extend(torch.cat([tokens, pad]), cache, table, _i32([2] * 3), start, max_q)
        assert bool(torch.isfinite(out).all())
        for layer in range(cfg.n_layers):
            assert not bool(rec.o[layer].view(40, -1)[6:].any())
    rec.close()


def test_bad_pages_are_reported():
    import computd_b200 as cb

    cfg, model = _model()
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    table[1, 0] = 24
    out = model.extend(_tokens(cfg)[:, :5].reshape(-1), cache, table, _i32([5] * 3))
    assert bool(torch.isnan(out.view(3, 5, -1)[1]).any())
    assert not bool(torch.isnan(out.view(3, 5, -1)[0]).any())
    with pytest.raises(cb.DWAError):
        cache.check()
    cache.check()


def test_cache_read_brings_back_the_layer():
    cfg, model = _model()
    cache = model.new_cache(24, page_size=16)
    table = _table(cfg, cache)
    tokens = _tokens(cfg)
    model.extend(tokens.reshape(-1), cache, table, _i32([64] * 3))
    start = _i32([0, 64, 128, 192])
    slots, positions = cache.slots(table, _i32([64] * 3), start, 192)
    assert positions.tolist() == list(range(64)) * 3
    k, v = cache.read(1, slots)
    at = (slots // 16, slots % 16)
    assert torch.equal(k, cache.k[1][at[0], :, at[1]]) and torch.equal(v, cache.v[1][at[0], :, at[1]])
