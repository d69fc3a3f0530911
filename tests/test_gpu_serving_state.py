"""GPU: what the calls of a model share between row counts, streams and captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_captured_rows_workspace_is_the_graphs_own():
    """The row-stationary assembly's scratch inside a captured graph belongs to that graph: not to
    the stream (whose buffer is replaced when a larger call comes), nor to another graph."""
    from computd_b200 import assembler

    d, r, k, rows = 64, 2, 8, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    vectors = torch.randn((rows, 2 * d * r + d), device="cuda", generator=g).bfloat16()

    def inputs(M):
        return (torch.randn((M, d), device="cuda", generator=g).bfloat16(),
                torch.rand((M, k), device="cuda", generator=g),
                torch.randint(0, rows, (M, k), device="cuda", generator=g).int())

    def call(x):
        return assembler.lowrank_delta(*x, vectors, d, d, r, rows=True)

    seen = []
    make = assembler.lowrank_rows_workspace

    def noted(*a):
        ws = make(*a)
        seen.append(ws.data_ptr())
        return ws

    small, large, largest = inputs(40), inputs(400), inputs(4000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    assembler.lowrank_rows_workspace = noted
    try:
        with torch.cuda.stream(side):
            want = [call(small).clone(), call(large).clone()]
            torch.cuda.synchronize()
            for x in (small, large):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = call(x)
                graphs.append((graph, out))
    finally:
        assembler.lowrank_rows_workspace = make
    eager, captured = seen[:2], seen[2:]
    assert not set(eager) & set(captured) and captured[0] != captured[1]
    with torch.cuda.stream(side):  # the stream's buffer is replaced, its memory goes to others
        call(largest)
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]
        for _ in range(5):
            for graph, _ in graphs:
                graph.replay()
    torch.cuda.synchronize()
    assert all(bool((x == 255).all()) for x in junk)
    for (_, out), x in zip(graphs, want):
        assert torch.equal(out, x)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prompt(cfg, model, b, n, page_size=16):
    """A cache of one layout, a table and n tokens of b sequences, alike for the same arguments."""
    cache = model.new_cache(b * (-(-64 // page_size)), page_size=page_size)
    table = torch.arange(cache.n_pages, device="cuda").int().view(b, -1)
    ids = torch.randint(0, cfg.vocab, (b, n), device="cuda", generator=torch.Generator("cuda").manual_seed(b + n))
    return cache, table, ids.reshape(-1), _i32([n] * b)


@pytest.mark.parametrize("r", [0, 2])
def test_plans_are_few_and_their_own(r):
    """Chunks of every row count from 1 to 150 make eight plans and one of 256; with r > 0 each
    has keys of its own; a plan's status and the model's are read; closed plans are gone."""
    from test_gpu_lm_extend import _model

    cfg, model = _model(r=r, dh=16 if r else 32, layers=1)
    cache, table, ids, _ = _prompt(cfg, model, 3, 50)
    for n in range(1, 151):
        seqs = 1 if n <= 50 else 3
        new = [n] if seqs == 1 else [50, 50, n - 100] if n > 100 else [50, n - 50, 0]
        start = _i32([sum(new[:b]) for b in range(seqs + 1)])
        model.extend(ids[:n], cache, table[:seqs], _i32(new), start, 50)
    assert sorted(model._chunk_plans) == [1, 2, 4, 8, 16, 32, 64, 128, 256]
    keys = [p.keys.data_ptr() for p in model._chunk_plans.values()] + [model.retriever.keys.data_ptr()]
    assert len(set(keys)) == (len(keys) if r else 1)
    assert model.status() == 0
    plan = model._chunk_plans[64].retriever
    was, plan.status = plan.status, lambda: 7
    assert model.status() == 7
    plan.status = was
    cache.check()
    model.close()
    assert not model._chunk_plans


@pytest.mark.parametrize("r", [0, 2])
@pytest.mark.parametrize("T", [1, 3, 65, 127, 129, 190])
def test_padded_plans_give_the_same(r, T):
    """A chunk's retrieval over a plan of more rows is bit for bit that of a plan of its own, also
    where the rows behind it held other queries."""
    import computd_b200 as cb
    from test_gpu_lm_extend import _model

    from computd_b200.dwa_lm import ChunkPlan

    cfg, model = _model(r=r, dh=16 if r else 32, layers=1)
    keys = cb.new_normal(cfg.pool_rows, cfg.key_width, seed=5, stddev=cfg.key_width ** -0.5, device="cuda")
    g = torch.Generator("cuda").manual_seed(T)
    exact, padded = ChunkPlan(model._plan(T)), model._chunk_plan(T)
    for plan in (exact, padded):
        plan.keys.copy_(keys)
    padded(torch.randn((padded.retriever.M, cfg.key_width), device="cuda", generator=g).bfloat16())
    q = torch.randn((T, cfg.key_width), device="cuda", generator=g).bfloat16()
    for x, y in zip(exact(q), padded(q)):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.shape[0] == y.shape[0] == T and torch.equal(x, y)


@pytest.mark.parametrize("r", [0, 2])
def test_two_row_counts_on_two_streams(r):
    """A prompt's chunk and single tokens of other sequences at the same time: what each alone gives."""
    from test_gpu_lm_extend import _model

    cfg, model = _model(r=r, dh=16 if r else 32, layers=4)
    for blk in model.blocks[1:]:  # blocks whose keys differ: another block's are wrong
        blk.retrieval.W_Q.copy_(blk.retrieval.W_Q.roll(1, -1))
    work = [_prompt(cfg, model, 3, 60), _prompt(cfg, model, 2, 1), _prompt(cfg, model, 5, 7)]
    call = lambda w: model.extend(w[2], w[0], w[1], w[3])  # noqa: E731
    want = [call(w).clone() for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[] for _ in work]
    for _ in range(30):
        for w, s, out in zip(work, streams, got):
            with torch.cuda.stream(s):
                out.append(call(w))
    torch.cuda.synchronize()
    for x, out in zip(want, got):
        assert all(torch.equal(x, y) for y in out)
    assert model.status() == 0


def test_verify_with_a_lost_last_token():
    """A sequence whose last token is -1, among others: reported, -1, unchanged; the others as alone;
    captured and replayed it does the same."""
    import computd_b200 as cb
    from test_gpu_lm_extend import _model

    cfg, model = _model(seed=4)
    cache, table, ids, lengths = _prompt(cfg, model, 3, 20)
    model.extend(ids, cache, table, lengths)
    g = torch.Generator("cuda").manual_seed(1)
    drafts = torch.randint(0, cfg.vocab, (3, 4), device="cuda", generator=g).int()
    u, r = torch.zeros((3, 4), device="cuda"), torch.rand(3, device="cuda", generator=g)
    good = _i32([3, 9, 60])
    want = [t.clone() for t in model.verify(good, drafts, None, u, r, cache, table, lengths)]
    cache.check()
    last = _i32([3, -1, 60])
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = model.verify(last, drafts, None, u, r, cache, table, lengths)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                again = model.verify(last, drafts, None, u, r, cache, table, lengths)
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for (accepted, tokens, new) in (got, again):
            for b in (0, 2):
                assert all(torch.equal(x[b], y[b]) for x, y in zip((accepted, tokens, new), want))
            assert accepted[1] == 0 and tokens[1].tolist() == [-1] * 5 and new[1] == 20
        with pytest.raises(cb.DWAError):
            cache.check()
        cache.check()


def test_an_output_that_does_not_fit_is_torchs_own_error():
    """A server that makes room and tries again catches torch.OutOfMemoryError."""
    import computd_b200 as cb

    cache = torch.zeros((1, 64, 16, 128), dtype=torch.bfloat16, device="cuda")
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    slots = torch.full((1 << 18,), -1, dtype=torch.int64, device="cuda")  # 8 GB of keys and values
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (4 << 30)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            cb.kv_cache_read(cache, cache, slots)
        k, v = cb.kv_cache_read(cache, cache, slots[:64])
        assert not bool(k.any()) and not bool(v.any())
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


@pytest.mark.parametrize("first,then", [(True, False), (False, True)])
def test_steps_in_and_out_of_inference_mode(first, then):
    """Plans, caches and their padded rows made in one mode serve in the other."""
    from test_gpu_lm_extend import _model

    cfg, model = _model(r=2, dh=16, layers=2)
    out = []
    with torch.inference_mode(first):
        cache, table, ids, lengths = _prompt(cfg, model, 3, 20)
    for mode in (first, then, first):
        with torch.inference_mode(mode):
            out.append(model.extend(ids, cache, table, lengths).clone())
            drafts = torch.full((3, 2), 5, dtype=torch.int32, device="cuda")
            u, r = torch.zeros((3, 2), device="cuda"), torch.zeros(3, device="cuda")
            model.verify(_i32([1, 2, 3]), drafts, None, u, r, cache, table, lengths)
            cache.check()
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
