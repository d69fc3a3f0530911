"""The operators of a serving step whose drafted tokens form a tree, and the cases they are
measured on.

A tree is n nodes per sequence, parents before children; node 0 is the sequence's newest token, the
others are drafts.  In the order a step makes the calls:

* ``tree_masks``: from every node's parent, the nodes that it sees (itself and its ancestors, as
  bits) and its depth.
* ``kv_cache_append``: the nodes' (or a prompt's) queries and keys rotated for their positions, keys
  and values into a paged cache, as bf16 or as e4m3 with one f32 scale per (token, head).
* ``paged_tree_attention``: every node over the tokens cached before the tree and the nodes
  its mask names.
* ``verify_tree``: from node 0 on, a token is drawn from the node's row of the target's probabilities
  with a given uniform number; where a child has it the walk goes on there, else it ends.
* ``kv_cache_keep``: the tokens of the path that stood move to the places behind the
  sequence's earlier ones, in every layer.

``run`` computes them in plain torch operations, or with ``own`` set by this package's kernels.
Heads, widths and vocabularies are those of the package's language model configurations (6 x 64,
16 x 80, 16 x 128, 32 x 128; 32000 and 64400 tokens), and grouped heads (32 over 8).
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


def listed():
    return [
        # the plan of one sequence's tree: latency
        dict(name="masks_one", op="masks", batch=1, new_lo=16, new_hi=16, deep=False),
        # plans of ragged trees for a large batch
        dict(name="masks_batch", op="masks", batch=64, new_lo=33, new_hi=128, deep=True),
        # one layer's append of a step with small trees, 8-bit cache, heads of 80: latency
        dict(name="append_step", op="append", kind="e4m3", heads=16, kv_heads=16, dim=80, page=32,
             tokens=64, pages=40, positions=2048),
        # a prompt of grouped heads into the bf16 cache, at far positions
        dict(name="append_prompt", op="append", kind="bf16", heads=32, kv_heads=8, dim=128, page=64,
             tokens=8191, pages=140, positions=32768),
        # small trees of the small character model: 16 sequences, everything is latency
        dict(name="attend_small", op="attend", kind="bf16", heads=6, kv_heads=6, dim=64, page=16,
             batch=16, new_lo=8, new_hi=16, ctx_lo=20, ctx_hi=256, deep=False),
        # trees of up to 32 nodes of the 1B model over a bf16 cache
        dict(name="attend_1b", op="attend", kind="bf16", heads=16, kv_heads=16, dim=128, page=64,
             batch=16, new_lo=20, new_hi=32, ctx_lo=300, ctx_hi=4096, deep=False),
        # up to 64 nodes over long 8-bit contexts with grouped heads
        dict(name="attend_long", op="attend", kind="e4m3", heads=32, kv_heads=8, dim=128, page=64,
             batch=16, new_lo=33, new_hi=64, ctx_lo=2000, ctx_hi=16384, deep=False),
        # the reference layout's heads of 80, ragged deep trees, short 8-bit contexts
        dict(name="attend_80", op="attend", kind="e4m3", heads=16, kv_heads=16, dim=80, page=32,
             batch=24, new_lo=5, new_hi=40, ctx_lo=50, ctx_hi=1500, deep=True),
        # one sequence's tree: the walk's latency
        dict(name="verify_one", op="verify", vocab=32000, batch=1, new_lo=16, new_hi=16, depth=5,
             deep=False),
        # trees of many sequences over the larger vocabulary
        dict(name="verify_batch", op="verify", vocab=64400, batch=32, new_lo=20, new_hi=32, depth=8,
             deep=False),
        # the small character model's accepted paths: 6 layers, latency
        dict(name="keep_small", op="keep", kind="bf16", layers=6, kv_heads=6, dim=64, page=16, batch=16,
             new=16, depth=5, ctx=100),
        # 12 layers of the 1B model in 8 bits, 32 sequences, long paths
        dict(name="keep_1b", op="keep", kind="e4m3", layers=12, kv_heads=16, dim=128, page=64, batch=32,
             new=64, depth=12, ctx=200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "verify", "verify", "keep", "masks"])
    if op == "masks":
        hi = _log(rng, 12, 128)
        return dict(op=op, batch=_log(rng, 1, 64), new_lo=hi // 3, new_hi=hi,
                    deep=rng.random() < 0.5)
    if op == "verify":
        hi = _log(rng, 2, 32)
        return dict(op=op, vocab=rng.choice([65, 32000, 64400, _log(rng, 65, 64400)]),
                    batch=_log(rng, 1, 32), new_lo=max(1, hi // 2), new_hi=hi, depth=rng.randint(1, 8),
                    deep=rng.random() < 0.5)
    kind = rng.choice(["bf16", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 80, 128])
    heads, kv_heads = rng.choice([(6, 6), (16, 16), (32, 32), (32, 8), (16, 2)])
    if op == "append":
        tokens = _log(rng, 1, 8000 if heads + 2 * kv_heads <= 48 else 4000)
        return dict(op=op, kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, tokens=tokens,
                    pages=-(-tokens // page) + rng.randint(1, 40), positions=_log(rng, 64, 100000))
    if op == "keep":
        depth = rng.randint(1, 12)
        return dict(op=op, kind=kind, layers=rng.randint(1, 12), kv_heads=min(kv_heads, 16), dim=dim,
                    page=page, batch=_log(rng, 1, 32), new=rng.randint(2 * depth + 2, 64), depth=depth,
                    ctx=rng.randint(1, 200))
    hi = _log(rng, 2, 128)
    batch = _log(rng, 1, 24)
    # no more cached vectors, and no more scores, than the largest listed cases have
    ctx_hi = min(_log(rng, 40, 16384), 16 * 16384 * 8 // (batch * kv_heads),
                 16 * 64 * 32 * 16384 // (batch * hi * heads))
    ctx_hi = max(ctx_hi, hi)
    return dict(op=op, kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch,
                new_lo=max(1, hi // rng.choice([1, 2, 5])), new_hi=hi,
                ctx_lo=max(hi, ctx_hi // rng.choice([1, 3, 20])), ctx_hi=ctx_hi, deep=rng.random() < 0.5)


def _trees(case, seed=0):
    """Every sequence's parents, -1 for node 0.  How many nodes they have is the case's alone, not the
    seed's."""
    sizes, rng = random.Random(11), random.Random(seed)
    got = []
    for b in range(case["batch"]):
        n = case["new_hi"] if b == 0 else sizes.randint(case["new_lo"], case["new_hi"])
        parents = [-1]
        for i in range(1, n):
            if case["deep"]:  # mostly chains, with side branches
                parents.append(i - 1 if rng.random() < 0.7 else rng.randrange(i))
            else:  # level by level, two to three children each
                parents.append(rng.randint(max(0, (i - 1) // 3), (i - 1) // 2))
        got.append(parents)
    return got


def _seen(parents):
    """For every node the set of itself and its ancestors, as bits."""
    got = []
    for i, p in enumerate(parents):
        got.append((1 << i) | (got[p] if p >= 0 else 0))
    return got


def _contexts(case):
    rng = random.Random(7)
    return [case["ctx_hi"] if b == 0 else rng.randint(case["ctx_lo"], case["ctx_hi"])
            for b in range(case["batch"])]


def _paths(case):
    """Every sequence's path (node numbers, node 0 first): a node either has its place already or lies
    behind all places, so that a second pass over the same state moves the same again."""
    rng = random.Random(5)
    got = []
    for b in range(case["batch"]):
        length = case["depth"] if b == 0 else rng.randint(0, case["depth"])
        still = rng.randint(0, min(2, length))
        got.append(list(range(still + 1))
                   + sorted(rng.sample(range(case["depth"] + 1, case["new"]), length - still)))
    return got


def work(case):
    op = case["op"]
    if op == "masks":
        nodes = sum(len(t) for t in _trees(case))
        return {"bytes": nodes * (4 + 8 * -(-case["new_hi"] // 64) + 4), "flops": nodes}
    if op == "verify":
        # the least a walk reads is one row of the vocabulary per sequence
        return {"bytes": case["batch"] * (case["vocab"] * 4 + (case["depth"] + 1) * 12) + 8 * case["new_hi"],
                "flops": case["batch"] * case["vocab"] * 2}
    d = case["dim"]
    row = d + 4 if case["kind"] == "e4m3" else 2 * d
    if op == "append":
        t, hq, hk = case["tokens"], case["heads"], case["kv_heads"]
        return {"bytes": t * (hq * 4 * d + 2 * hk * (2 * d + row) + 16) + min(t, case["positions"]) * 4 * d,
                "flops": t * (hq + hk) * 3 * d + t * 2 * hk * d}
    if op == "keep":
        moved = sum(sum(i != p for i, p in enumerate(path)) for path in _paths(case))
        return {"bytes": case["layers"] * moved * case["kv_heads"] * 2 * row * 2 + 64 * case["batch"], "flops": 0}
    nodes = cached = pairs = 0
    for parents, ctx in zip(_trees(case), _contexts(case)):
        nodes += len(parents)
        cached += ctx
        pairs += len(parents) * (ctx - len(parents)) + sum(bin(m).count("1") for m in _seen(parents))
    return {"bytes": 2 * nodes * case["heads"] * d * 2 + 2 * cached * case["kv_heads"] * row
            + 4 * -(-cached // case["page"]) + 8 * nodes * -(-case["new_hi"] // 64),
            "flops": 4 * case["heads"] * d * pairs}


def _quantise(x):
    """e4m3 codes and f32 scales of x [..., d]."""
    x = x.float()
    # a divisor on the device: one in the program would be turned into a product with 1 / 448
    scale = torch.clamp(x.abs().amax(-1) / torch.full((), E4M3_MAX, device=x.device), min=MIN_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _filled(case, gen, *pages):
    """A cache of these pages (or layers and pages) with keys and values in it."""
    shape = (*pages, case["kv_heads"], case["page"], case["dim"])
    got = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
        if case["kind"] == "e4m3":
            # heads of unlike size, as projections give them
            x = x * torch.logspace(-1, 1, case["kv_heads"], device="cuda", dtype=torch.bfloat16)[:, None, None] \
                if name == "v" else x
            got[name + "_cache"], got[name + "_scale"] = _quantise(x)
        else:
            got[name + "_cache"], got[name + "_scale"] = x, None
    return got


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(s, case, gen, contexts):
    """Pages of `contexts` tokens for every sequence, in no order, and a cache of them."""
    used = [-(-ctx // case["page"]) for ctx in contexts]
    total = sum(used) + 3
    s.update(_filled(case, gen, *([case["layers"], total] if case["op"] == "keep" else [total])))
    free = torch.randperm(total, generator=gen, device="cuda").int()
    s["table"] = torch.zeros((len(used), max(used)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        s["table"][b, :n] = free[at:at + n]
        at += n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    op = case["op"]
    s = {"op": op, "case": case}
    if op == "append":
        s.update(_filled(case, gen, case["pages"]))
        T, H, Hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s["slots"] = torch.randperm(case["pages"] * case["page"], generator=gen, device="cuda")[:T]
        # queries, keys and values in place in the projection's rows
        qkv = torch.randn((T, (H + 2 * Hk) * d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"] = qkv[:, :H * d].view(T, H, d)
        s["k"] = qkv[:, H * d:(H + Hk) * d].view(T, Hk, d)
        s["v"] = qkv[:, (H + Hk) * d:].view(T, Hk, d)
        # the model's rotation tables, by position; the tokens' positions follow one another
        angle = torch.outer(torch.arange(case["positions"], device="cuda", dtype=torch.float64),
                            10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        first = order.randrange(max(1, case["positions"] - T))
        s["positions"] = (first + torch.arange(T, device="cuda")) % case["positions"]
        return s
    if op == "keep":
        paths = _paths(case)
        order.shuffle(paths)
        start = [order.randint(0, case["ctx"]) for _ in paths]
        _tables(s, case, gen, [case["ctx"] + case["new"]] * len(paths))
        s["start"], s["kept"] = _i32(start), _i32([len(p) - 1 for p in paths])
        s["path"] = _i32([p + [-1] * (case["depth"] + 1 - len(p)) for p in paths])
        return s
    trees = _trees(case, seed)
    order.shuffle(trees)
    new = [len(t) for t in trees]
    s["q_start"] = _i32([sum(new[:b]) for b in range(len(new) + 1)])
    s["max_q"] = max(new)
    s["parents"] = _i32([p for t in trees for p in t])
    if op == "masks":
        return s
    if op == "verify":
        T, V = sum(new), case["vocab"]
        s["target"] = torch.softmax(4.0 * torch.randn((T, V), generator=gen, device="cuda"), -1)
        # a drafter near the target proposes distinct tokens below every node
        child, most = [], 1
        for t in trees:
            count = [0] * len(t)
            for p in t:
                child.append(count[p] if p >= 0 else 0)
                if p >= 0:
                    count[p] += 1
            most = max(most, *count)
        proposed = torch.multinomial(s["target"], most, generator=gen).int()
        row = [0 if p < 0 else base + p
               for t, base in zip(trees, s["q_start"].tolist()) for p in t]
        s["tokens"] = proposed[torch.tensor(row, device="cuda"), torch.tensor(child, device="cuda")].contiguous()
        s["u"] = torch.rand((len(new), case["depth"] + 1), generator=gen, device="cuda")
        return s
    contexts = _contexts(case)
    order.shuffle(contexts)
    contexts = [max(c, n) for c, n in zip(contexts, new)]
    _tables(s, case, gen, contexts)
    s["lengths"] = _i32(contexts)
    words = -(-s["max_q"] // 64)
    bits = [m for t in trees for m in _seen(t)]
    signed = lambda x: x - (1 << 64) if x >> 63 else x  # noqa: E731
    s["mask"] = torch.tensor([[signed((m >> (64 * w)) & ((1 << 64) - 1)) for w in range(words)] for m in bits],
                             device="cuda")
    s["q"] = torch.randn((sum(new), case["heads"], case["dim"]), generator=gen, device="cuda",
                         dtype=torch.bfloat16)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"masks": _masks, "append": _append, "attend": _attend, "verify": _verify, "keep": _keep}[s["op"]](s)


def _caches(s):
    return [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None]


def _run_own(s):
    import computd_b200 as cb

    if s["op"] == "masks":
        return cb.tree_masks(s["parents"], q_start=s["q_start"], max_q=s["max_q"])
    if s["op"] == "append":
        q = cb.kv_cache_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"],
                               s["slots"], positions=s["positions"], k_scale=s["k_scale"],
                               v_scale=s["v_scale"])
        return [q, *_caches(s)]
    if s["op"] == "attend":
        return cb.paged_tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                       s["mask"], q_start=s["q_start"], max_q=s["max_q"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["op"] == "verify":
        return cb.verify_tree(s["target"], s["tokens"], s["parents"], s["u"], q_start=s["q_start"])
    cb.kv_cache_keep(s["k_cache"], s["v_cache"], s["table"], s["start"], s["path"], s["kept"],
                     k_scale=s["k_scale"], v_scale=s["v_scale"])
    return _caches(s)


def _sequence(s, rows):
    """The sequence of every packed row."""
    start = s["q_start"].long()
    row = torch.arange(rows, device=start.device)
    return torch.searchsorted(start, row, right=True) - 1, row


def _masks(s):
    parents = s["parents"].long()
    T = parents.shape[0]
    seq, row = _sequence(s, T)
    base = s["q_start"].long()[seq]
    i = row - base
    words = torch.arange(-(-s["max_q"] // 64), device=row.device)
    mask = torch.where(words == (i // 64)[:, None], torch.ones_like(i)[:, None] << (i % 64)[:, None], 0)
    at = torch.where(parents >= 0, base + parents, -1)
    # every node takes what its ancestor sees, an ancestor twice as far each time
    for _ in range(max(s["max_q"] - 1, 0).bit_length()):
        some, up = at >= 0, at.clamp(min=0)
        mask = torch.where(some[:, None], mask | mask[up], mask)
        at = torch.where(some, at[up], -1)
    depth = ((mask[..., None] >> torch.arange(64, device=row.device)) & 1).sum((1, 2)) - 1
    return mask, depth.int()


def _append(s):
    def turned(x):
        c, sn = (s[n][s["positions"]][:, None] for n in ("cos", "sin"))
        x1, x2 = x.float()[..., 0::2], x.float()[..., 1::2]
        return torch.cat([x1 * c - x2 * sn, x1 * sn + x2 * c], -1)

    page = s["k_cache"].shape[2]
    at, off = s["slots"] // page, s["slots"] % page
    for name, x in (("k", turned(s["k"])), ("v", s["v"].float())):  # the two halves of the cache
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if scale is None:
            cache[at, :, off] = x.to(torch.bfloat16)
        else:
            codes, scales = _quantise(x)
            cache.view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            scale[at, :, off] = scales
    return [turned(s["q"]).to(torch.bfloat16), *_caches(s)]


def _attend(s):
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].long()
    T, heads, d = q.shape
    B, pages = table.shape
    _, kv_heads, page, _ = s["k_cache"].shape
    q_start = s["q_start"].long()
    new = q_start[1:] - q_start[:-1]
    # queries as [B, kv head, group * node, d]
    j = torch.arange(s["max_q"], device=q.device)
    rows = (q_start[:-1, None] + j).clamp(max=T - 1)
    group = heads // kv_heads
    qp = q[rows].float().view(B, -1, kv_heads, group, d).permute(0, 2, 3, 1, 4).reshape(B, kv_heads, -1, d)

    def dense(cache, scale):
        x = cache[table].float()
        if scale is not None:
            x = x * scale[table][..., None]
        return x.transpose(1, 2).reshape(B, kv_heads, pages * page, d)

    scores = torch.matmul(qp, dense(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * d ** -0.5
    at = torch.arange(pages * page, device=q.device)
    node = at - (lengths - new)[:, None]  # of the tree, from 0 on
    word = (node // 64).clamp(0, s["mask"].shape[1] - 1)
    seen = torch.gather(s["mask"][rows], 2, word[:, None].expand(-1, s["max_q"], -1))
    open_ = (node < 0)[:, None] | ((node < new[:, None])[:, None] & (((seen >> (node % 64)[:, None]) & 1) == 1))
    open_ = open_[:, None, None].expand(B, 1, group, -1, -1).reshape(B, 1, -1, pages * page)
    scores = scores.masked_fill(~open_, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, dense(s["v_cache"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    out = out.view(B, kv_heads, group, -1, d).permute(0, 3, 1, 2, 4).reshape(B, -1, heads, d)
    seq, row = _sequence(s, T)
    return out[seq, row - q_start[seq]].to(q.dtype)


def _verify(s):
    p, start = s["target"], s["q_start"].long()
    B, steps = s["u"].shape
    T, V = p.shape
    seq, row = _sequence(s, T)
    b = torch.arange(B, device=p.device)
    node = torch.zeros(B, dtype=torch.long, device=p.device)
    going = torch.ones(B, dtype=torch.bool, device=p.device)
    kept = torch.zeros(B, dtype=torch.long, device=p.device)
    tokens = torch.full((B, steps), -1, dtype=torch.int32, device=p.device)
    path = torch.full((B, steps), -1, dtype=torch.int32, device=p.device)
    inner = row - start[seq]
    for i in range(steps):
        # running sums next to a uniform number: in 64 bits, so that borders fall alike
        run_ = p[start[:-1] + node].double().cumsum(-1)
        token = (run_ <= s["u"][:, i].double()[:, None] * run_[:, -1:]).sum(-1).clamp(max=V - 1)
        tokens[:, i] = torch.where(going, token, -1).int()
        path[:, i] = torch.where(going, node, -1).int()
        fits = ((s["parents"] == node[seq]) & (s["tokens"] == token[seq]) & (inner > 0))
        child = torch.full((B,), T, device=p.device).scatter_reduce(0, seq, torch.where(fits, inner, T), "amin")
        going = going & (child < T) & (i + 1 < steps)
        kept = kept + going
        node = torch.where(going, child, 0)
    return kept.int(), tokens, path


def _keep(s):
    page = s["k_cache"].shape[3]
    path = s["path"].long()
    place = torch.arange(path.shape[1], device=path.device)
    b, i = ((place <= s["kept"][:, None]) & (path != place)).nonzero(as_tuple=True)
    old, new = s["start"][b] + path[b, i], s["start"][b] + i
    old_page, new_page = s["table"][b, old // page].long(), s["table"][b, new // page].long()
    for x in _caches(s):
        x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
        x[:, new_page, :, new % page] = x[:, old_page, :, old % page].clone()
    return _caches(s)


def exact(case, seed):
    op = case["op"]
    if op in ("masks", "keep"):  # nothing is rounded: whole numbers, and values that move
        return None
    s = prepare(case, seed)
    if op == "verify":
        start = s["q_start"].tolist()
        parents, drafted = s["parents"].tolist(), s["tokens"].tolist()
        kept, tokens, path = [], [], []
        for b in range(case["batch"]):
            node, got, way = 0, [], []
            while True:
                c = torch.cumsum(s["target"][start[b] + node].double().cpu(), 0)
                goal = torch.tensor([float(s["u"][b, len(got)]) * float(c[-1])], dtype=torch.float64)
                t = min(int(torch.searchsorted(c, goal, right=True)), case["vocab"] - 1)
                got.append(t)
                way.append(node)
                below = [i for i in range(1, start[b + 1] - start[b])
                         if parents[start[b] + i] == node and drafted[start[b] + i] == t]
                if not below or len(got) > case["depth"]:
                    break
                node = below[0]
            kept.append(len(got) - 1)
            tokens.append(got + [-1] * (case["depth"] + 1 - len(got)))
            path.append(way + [-1] * (case["depth"] + 1 - len(way)))
        return tuple(torch.tensor(x, dtype=torch.int32) for x in (kept, tokens, path))
    slots_of = lambda x: x.transpose(1, 2).flatten(0, 1)  # noqa: E731  [slot, head, ...]
    if op == "append":
        c, sn = (s[n].double()[s["positions"]][:, None] for n in ("cos", "sin"))

        def turned(x):
            even, odd = x.double().unflatten(-1, (-1, 2)).unbind(-1)
            return torch.cat([even * c - odd * sn, even * sn + odd * c], -1)

        pages, heads, page, d = s["k_cache"].shape
        caches, scales = [], []
        for name, x in (("k", turned(s["k"])), ("v", s["v"].double())):
            cache = slots_of(s[name + "_cache"].double()).clone()
            if case["kind"] == "e4m3":
                scale = (x.abs().amax(-1) / E4M3_MAX).clamp(min=MIN_SCALE).float()
                y = (x / scale[..., None].double()).float().double()  # the format's quotient has 32 bits
                # the nearest multiple of the spacing at its size, ties to even
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                x = (torch.round(y / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
                held = slots_of(s[name + "_scale"][..., None].double())[..., 0].clone()
                held[s["slots"]] = scale.double()
                scales.append(held.view(pages, page, heads).transpose(1, 2))
            cache[s["slots"]] = x
            caches.append(cache.view(pages, page, heads, d).transpose(1, 2))
        return [turned(s["q"]), *caches, *scales]
    q, start = s["q"].double(), s["q_start"].tolist()
    parents = s["parents"].tolist()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, length in enumerate(s["lengths"].tolist()):
        ids = s["table"][b].long()[:-(-length // case["page"])]
        rows = slice(start[b], start[b + 1])
        n = start[b + 1] - start[b]
        hidden = torch.ones((n, n), dtype=torch.bool)
        for i in range(n):  # up to the root
            j = i
            while j >= 0:
                hidden[i, j] = False
                j = parents[start[b] + j]
        hidden = torch.cat([torch.zeros((n, length - n), dtype=torch.bool), hidden], 1).cuda()
        for h in range(case["kv_heads"]):
            def column(name):
                x = s[name + "_cache"][ids, h].double()
                if s[name + "_scale"] is not None:
                    x = x * s[name + "_scale"][ids, h].double()[..., None]
                return x.flatten(0, 1)[:length]

            k, v = column("k"), column("v")
            for g in range(h * group, (h + 1) * group):
                w = (q[rows, g] @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                out[rows, g] = torch.softmax(w, -1) @ v
    return out
