"""The serving operators of the language model and the cases they are measured on.

Four calls, in the order a serving step makes them:

* ``kv_cache_write``: new tokens' keys and values into a paged cache, as bf16 or
  as e4m3 with one f32 scale per (token, head): scale = max(amax / 448, 2^-126),
  code = e4m3(x / scale).
* ``paged_attention``: a chunk of new tokens of every sequence (one token, a few
  drafted ones, a long prompt's piece) over that cache, causal at the
  chunk's end: token j of n attends to the cache's first length - n + j + 1 tokens.
* ``verify_drafts``: drafted tokens held against the target's probabilities with
  given uniform numbers: draft i stands if u_i q_i(x_i) < p_i(x_i); the first that
  falls is replaced by a draw from max(p - q, 0), or the token after the last by one from p.
* ``kv_cache_read``: cached tokens back as bf16 rows.

``run`` computes them in plain torch operations, or with ``own`` set by this
package's kernels.  Heads, widths and vocabularies are those of the package's
language model configurations (6 x 64, 16 x 80, 16 x 128, 32 x 128; 32000 and 64400
tokens), and grouped heads (32 over 8).
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


def listed():
    return [
        # one decoding step of the small character model: 16 sequences, everything is latency
        dict(name="attend_decode_small", op="attend", kind="bf16", heads=6, kv_heads=6, dim=64, page=16,
             batch=16, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=256),
        # one decoding step of the 1B model, 64 ragged sequences, bf16 cache
        dict(name="attend_decode_1b", op="attend", kind="bf16", heads=16, kv_heads=16, dim=128, page=64,
             batch=64, new_lo=1, new_hi=1, ctx_lo=90, ctx_hi=2048),
        # long contexts with grouped heads in an 8-bit cache: the bytes of the cache are all that counts
        dict(name="attend_decode_long", op="attend", kind="e4m3", heads=32, kv_heads=8, dim=128, page=64,
             batch=32, new_lo=1, new_hi=1, ctx_lo=4000, ctx_hi=16384),
        # drafted tokens of the reference layout's model (heads of 80), 1 to 6 per sequence
        dict(name="attend_drafts", op="attend", kind="e4m3", heads=16, kv_heads=16, dim=80, page=32,
             batch=24, new_lo=1, new_hi=6, ctx_lo=33, ctx_hi=1024),
        # a long prompt of the 7B model in pieces: the second piece over a filled cache, tensor-bound
        dict(name="attend_chunk_7b", op="attend", kind="bf16", heads=32, kv_heads=32, dim=128, page=128,
             batch=2, new_lo=2048, new_hi=2048, ctx_lo=4096, ctx_hi=8192),
        # uneven pieces of three prompts with grouped heads over an 8-bit cache
        dict(name="attend_chunk_ragged", op="attend", kind="e4m3", heads=32, kv_heads=8, dim=128, page=64,
             batch=3, new_lo=131, new_hi=1000, ctx_lo=1500, ctx_hi=9001),
        # one decoding step's keys and values into the 8-bit cache
        dict(name="write_step", op="write", kind="e4m3", kv_heads=16, dim=128, page=64, tokens=64,
             pages=160),
        # a prompt of the 7B model into the 8-bit cache
        dict(name="write_prompt", op="write", kind="e4m3", kv_heads=32, dim=128, page=64, tokens=8191,
             pages=140),
        # a short prefix back from the 8-bit cache
        dict(name="read_prefix", op="read", kind="e4m3", kv_heads=16, dim=80, page=32, tokens=333,
             pages=64),
        # a whole context back, for a layer that wants it dense
        dict(name="read_context", op="read", kind="e4m3", kv_heads=32, dim=128, page=64, tokens=16384,
             pages=300),
        # four drafts for one sequence: latency
        dict(name="verify_one", op="verify", vocab=32000, batch=1, drafts=4),
        # seven drafts for each of 64 sequences over the larger vocabulary
        dict(name="verify_batch", op="verify", vocab=64400, batch=64, drafts=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "verify"])
    if op == "verify":
        return dict(op=op, vocab=rng.choice([65, 32000, 64400, _log(rng, 65, 64400)]),
                    batch=_log(rng, 1, 64), drafts=rng.randint(1, 7))
    kind = rng.choice(["bf16", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 80, 128])
    if op != "attend":
        heads = rng.choice([6, 8, 16, 32])
        tokens = _log(rng, 1, 8000)
        return dict(op=op, kind=kind, kv_heads=heads, dim=dim, page=page, tokens=tokens,
                    pages=-(-tokens // page) + rng.randint(1, 40))
    heads, kv_heads = rng.choice([(6, 6), (16, 16), (32, 32), (32, 8), (16, 2)])
    form = rng.choice(["one", "drafts", "chunk"])
    batch = _log(rng, 1, 48) if form != "chunk" else rng.randint(1, 4)
    new_hi = {"one": 1, "drafts": rng.randint(2, 8), "chunk": _log(rng, 17, 1500)}[form]
    new_lo = new_hi if rng.random() < 0.3 else 1 if form != "chunk" else max(1, new_hi // 4)
    # no more cache than the largest listed cases read
    ctx_hi = min(_log(rng, 16, 16384), 32 * 16384 * 8 // (batch * kv_heads))
    if form == "chunk":
        ctx_hi = min(ctx_hi, 8000)
    ctx_hi = max(ctx_hi, new_hi)
    ctx_lo = max(new_hi, ctx_hi // rng.choice([1, 3, 20]))
    return dict(op=op, kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch,
                new_lo=new_lo, new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi)


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of every sequence: the case's alone, not the seed's."""
    rng = random.Random(7)
    got = []
    for b in range(case["batch"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        ctx = rng.randint(case["ctx_lo"], case["ctx_hi"])
        got.append((n, max(n, case["ctx_hi"] if b == 0 else ctx)))
    return got


def work(case):
    d = case.get("dim", 0)
    row = d * (1 if case.get("kind") == "e4m3" else 2) + (4 if case.get("kind") == "e4m3" else 0)
    if case["op"] == "verify":
        # a rejected sequence reads its row of p and of q; the tests of the drafts are a few values
        return {"bytes": case["batch"] * (2 * case["vocab"] * 4 + case["drafts"] * 16 + 12),
                "flops": case["batch"] * case["vocab"] * 3}
    if case["op"] in ("write", "read"):
        vectors = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": vectors * (2 * d + row) + 8 * case["tokens"], "flops": vectors * d * 3}
    rows = cached = pairs = 0
    for n, ctx in _lengths(case):
        rows += n
        cached += ctx
        pairs += n * (ctx - n) + n * (n + 1) // 2
    return {"bytes": 2 * rows * case["heads"] * d * 2 + 2 * cached * case["kv_heads"] * row
            + 4 * -(-cached // case["page"]),
            "flops": 4 * case["heads"] * d * pairs}


def _quantise(x):
    """e4m3 codes and f32 scales of x [..., d]."""
    x = x.float()
    # a divisor on the device: one in the program would be turned into a product with 1 / 448
    scale = torch.clamp(x.abs().amax(-1) / torch.full((), E4M3_MAX, device=x.device), min=MIN_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _filled(case, gen, pages):
    """A cache of `pages` pages with keys and values in it."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
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


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    s = {"op": case["op"], "case": case}
    if case["op"] == "verify":
        B, K, V = case["batch"], case["drafts"], case["vocab"]
        logits = 2.0 * torch.randn((B, K + 1, V), generator=gen, device="cuda")
        near = logits[:, :K] + 0.5 * torch.randn((B, K, V), generator=gen, device="cuda")
        s["target"], s["draft"] = torch.softmax(logits, -1), torch.softmax(near, -1)
        s["tokens"] = torch.multinomial(s["draft"].view(B * K, V), 1, generator=gen).view(B, K).int()
        s["accept_u"] = torch.rand((B, K), generator=gen, device="cuda")
        s["sample_u"] = torch.rand((B,), generator=gen, device="cuda")
        # drafters stop early at times
        s["lengths"] = torch.tensor([K if b % 3 else order.randint(0, K) for b in range(B)],
                                    dtype=torch.int32, device="cuda")
        return s
    H, d, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] in ("write", "read"):
        s.update(_filled(case, gen, case["pages"]))
        T = case["tokens"]
        s["slots"] = torch.randperm(case["pages"] * page, generator=gen, device="cuda")[:T]
        if case["op"] == "write":
            # keys as the rotary embedding leaves them, values in place in the projection's rows
            s["k"] = torch.randn((T, H, d), generator=gen, device="cuda", dtype=torch.bfloat16)
            qkv = torch.randn((T, 3 * H * d), generator=gen, device="cuda", dtype=torch.bfloat16)
            s["v"] = qkv[:, 2 * H * d:].view(T, H, d)
        return s
    lengths = _lengths(case)
    order.shuffle(lengths)
    used = [-(-ctx // page) for _, ctx in lengths]
    s.update(_filled(case, gen, sum(used) + 3))
    free = torch.randperm(sum(used) + 3, generator=gen, device="cuda").int()
    s["table"] = torch.zeros((len(used), max(used)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        s["table"][b, :n] = free[at:at + n]
        at += n
    s["lengths"] = torch.tensor([ctx for _, ctx in lengths], dtype=torch.int32, device="cuda")
    new = [n for n, _ in lengths]
    start = [sum(new[:b]) for b in range(len(new) + 1)]
    s["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    s["max_q"] = max(new)
    s["q"] = torch.randn((start[-1], case["heads"], d), generator=gen, device="cuda", dtype=torch.bfloat16)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"attend": _attend, "write": _write, "read": _read, "verify": _verify}[s["op"]](s)


def _run_own(s):
    import computd_b200 as cb

    if s["op"] == "attend":
        return cb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                  q_start=s["q_start"], max_q=s["max_q"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"])
    if s["op"] == "write":
        cb.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                          v_scale=s["v_scale"])
        return [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None]
    if s["op"] == "read":
        return cb.kv_cache_read(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                                v_scale=s["v_scale"])
    return cb.verify_drafts(s["target"], s["tokens"], s["draft"], s["accept_u"], s["sample_u"],
                            draft_lengths=s["lengths"])


def _attend(s):
    q, table, lengths, q_start = s["q"], s["table"].long(), s["lengths"].long(), s["q_start"].long()
    T, heads, d = q.shape
    B, pages = table.shape
    _, kv_heads, page, _ = s["k_cache"].shape
    new = q_start[1:] - q_start[:-1]
    # queries as [B, kv head, group * token, d]
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
    last = (lengths - new)[:, None] + j
    open_ = at < torch.minimum(last + 1, lengths[:, None])[..., None]
    open_ = open_[:, None, None].expand(B, 1, group, -1, -1).reshape(B, 1, -1, pages * page)
    scores = scores.masked_fill(~open_, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, dense(s["v_cache"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    out = out.view(B, kv_heads, group, -1, d).permute(0, 3, 1, 2, 4).reshape(B, -1, heads, d)
    row = torch.arange(T, device=q.device)
    seq = torch.searchsorted(q_start, row, right=True) - 1
    return out[seq, row - q_start[seq]].to(q.dtype)


def _write(s):
    page = s["k_cache"].shape[2]
    at, off = s["slots"] // page, s["slots"] % page
    for name in ("k", "v"):  # the two halves of the cache
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if scale is None:
            cache[at, :, off] = s[name]
        else:
            codes, scales = _quantise(s[name])
            cache.view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            scale[at, :, off] = scales
    return [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None]


def _read(s):
    page = s["k_cache"].shape[2]
    at, off = s["slots"] // page, s["slots"] % page

    def back(cache, scale):
        if scale is None:
            return cache[at, :, off]
        return (cache.view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn).float()
                * scale[at, :, off][..., None]).to(torch.bfloat16)

    return back(s["k_cache"], s["k_scale"]), back(s["v_cache"], s["v_scale"])


def _verify(s):
    p, q, x, n = s["target"], s["draft"], s["tokens"].long(), s["lengths"].long()
    B, K, V = q.shape
    # products of two 24-bit fractions and running sums: in 64 bits, so that borders fall alike
    px = p[:, :K].gather(-1, x[..., None])[..., 0].double()
    qx = q.gather(-1, x[..., None])[..., 0].double()
    stands = (s["accept_u"].double() * qx < px) & (torch.arange(K, device=p.device) < n[:, None])
    kept = stands.long().cumprod(-1).sum(-1)
    b = torch.arange(B, device=p.device)
    target = p[b, kept].double()
    draft = q[b, kept.clamp(max=K - 1)].double()
    rest = torch.where((kept < n)[:, None], (target - draft).clamp(min=0), target)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, target)
    run_ = rest.cumsum(-1)
    token = (run_ <= s["sample_u"].double()[:, None] * run_[:, -1:]).sum(-1).clamp(max=V - 1)
    i = torch.arange(K + 1, device=p.device)
    padded = torch.cat([x, x[:, :1]], -1)
    tokens = torch.where(i < kept[:, None], padded, torch.where(i == kept[:, None], token[:, None], -1))
    return kept.int(), tokens.int()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        kept, tokens = [], []
        for b in range(case["batch"]):
            p, q, n = s["target"][b].double().cpu(), s["draft"][b].double().cpu(), int(s["lengths"][b])
            row, weight = [], None
            for i in range(n):
                x = int(s["tokens"][b, i])
                if not float(s["accept_u"][b, i]) * float(q[i, x]) < float(p[i, x]):
                    weight = torch.relu(p[i] - q[i])
                    break
                row.append(x)
            if weight is None or float(weight.sum()) <= 0:
                weight = p[len(row)]
            c = torch.cumsum(weight, 0)
            t = int(torch.searchsorted(c, torch.tensor([float(s["sample_u"][b]) * float(c[-1])],
                                                       dtype=torch.float64), right=True))
            kept.append(len(row))
            row.append(min(t, case["vocab"] - 1))
            tokens.append(row + [-1] * (case["drafts"] + 1 - len(row)))
        return torch.tensor(kept, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
    slots_of = lambda x: x.transpose(1, 2).flatten(0, 1)  # noqa: E731  [slot, head, ...]

    def values(name):
        x, scale = slots_of(s[name + "_cache"].double()), s[name + "_scale"]
        return x if scale is None else x * slots_of(scale[..., None].double())

    if case["op"] == "read":
        return values("k")[s["slots"]], values("v")[s["slots"]]
    if case["op"] == "write":
        pages, heads, page, d = s["k_cache"].shape
        caches, scales = [], []
        for name in ("k", "v"):
            x = s[name].double()
            cache = slots_of(s[name + "_cache"].double()).clone()
            if case["kind"] == "e4m3":
                scale = (x.abs().amax(-1) / E4M3_MAX).clamp(min=MIN_SCALE).float()
                y = x / scale[..., None].double()
                # the nearest multiple of the spacing at its size, ties to even
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                x = torch.round(y / step) * step
                held = slots_of(s[name + "_scale"][..., None].double())[..., 0].clone()
                held[s["slots"]] = scale.double()
                scales.append(held.view(pages, page, heads).transpose(1, 2))
            cache[s["slots"]] = x
            caches.append(cache.view(pages, page, heads, d).transpose(1, 2))
        return caches + scales
    q, start = s["q"].double(), s["q_start"].tolist()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, length in enumerate(s["lengths"].tolist()):
        ids = s["table"][b].long()[:-(-length // case["page"])]
        rows = slice(start[b], start[b + 1])
        n = start[b + 1] - start[b]
        for h in range(case["kv_heads"]):
            def column(name):
                x = s[name + "_cache"][ids, h].double()
                if s[name + "_scale"] is not None:
                    x = x * s[name + "_scale"][ids, h].double()[..., None]
                return x.flatten(0, 1)[:length]

            k, v = column("k"), column("v")
            for g in range(h * group, (h + 1) * group):
                w = q[rows, g] @ k.T / math.sqrt(case["dim"])
                w = w + torch.full_like(w, -math.inf).triu(length - n + 1)
                out[rows, g] = torch.softmax(w, -1) @ v
    return out
