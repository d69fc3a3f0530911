"""DWA language model forward — the call site of the retrieval path.

Mirrors the reference's ``DWAModel`` / ``DWABlock`` (src/model/dwa.py:77-216)
to measure the path inside a model (tokens/s).  Each block composes the
reference's own pieces in the reference's order (dwa.py:100-130):

    h = PartA(tokens)                                   parts.py:88-143
    for each block:
        h = attn(h)                                      dwa.py:101-102, parts.py:30-83
        z = query_proj(h)                                dwa.py:103
        alpha, idx = MultiAspectRetrieval(z, pool)       retrieval.py:131-181 (hybrid layout)
        h = WeightAssembler(h, alpha, idx, pool)         dwa.py:129, assembly.py:75-128
    logits = PartB(h)                                    parts.py:146-176

Retrieval (``MultiAspectRetrieval`` parameters W_Q [S, d_k, d], aspect_logits
and tau, retrieval.py:22-44): the per-position queries are projected per
aspect, L2-normalised and packed as [sqrt(w_s) q_s]_s (d = S d_k), so that one
dot product with the packed pool keys [sqrt(w_s) k_s]_s is hybrid_forward's
aspect-weighted score sum_s w_s <q_s, k_s> (retrieval.py:154-165); the fused
score + top-k kernel keeps the k best per position (retrieval.py:175) and
alpha = v / (sum v + 1e-8) (178).

The pool comes in one of two layouts:

* ``r > 0`` (the reference's own layout, configs/large_1b.py): pool vectors
  [N, D] hold [U (d r) | V (r d) | b (d)] rows (assembly.py:10-14).  Each
  block projects its pool keys from them with its own W_K [S, d_k, D]
  (retrieval.py:155-156: one tcgen05 launch per block and forward, as the
  reference's training forward recomputes them), and the WeightAssembler adds
  h_delta + b_delta = sum_j alpha_j (U_j (V_j h) + b_j) (assembly.py:104-128,
  ``dwa_lowrank_delta``) before LayerNorm(h + gamma (h W_base^T + b_base + .)).
* ``r == 0`` (the benchmark layouts: a synthetic [N, S d_k] key pool standing
  in for the cached packed keys, and value rows [N, d]): the retrieved value
  rows are the b vectors of the WeightAssembler formula, b_delta =
  sum_j alpha_j V_j (the gathered weighted sum, ``dwa_weighted_gather``), with
  no low-rank term.

The pool is shared by every block (dwa.py:182, 195) and optionally row-sharded
over a process group (one cross-shard merge per block, owner-computes value
sums).  Dense layers (attention, projections, PartA/PartB) are plain
torch/cuBLAS; retrieval, key projection, assembly delta and its LayerNorm
finish run in libdwa_b200.so.

``DWALM.extend`` is the same model over a paged key/value cache, for generation
(the reference runs whole windows for every token, src/training/trainer.py:258-338):
it takes the newest tokens of any number of sequences (prompts in pieces, single
tokens, drafted ones), writes their keys and values and attends to the pages with
``kv_cache``'s kernels.  ``DWALM.verify`` scores drafted tokens that way and
decides with ``verify_drafts`` which of them stand; ``DWALM.verify_tree`` does so for
trees of them, several candidates to a place.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .assembler import WeightAssembler
from .assembly import _check_values
from .kv_cache import PagedKVCache, tree_masks, verify_drafts, verify_tree
from .lm_ops import aspect_queries, rope_qk
from .retrieval import MultiAspectRetrieval, Retriever, project_keys_packed
from .tiled_topk import _as_bf16_rows


@dataclass(frozen=True)
class DWALMConfig:
    vocab: int
    d_model: int
    n_layers: int
    n_heads: int
    seq_len: int
    batch: int
    pool_rows: int
    top_k: int
    S: int                    # retrieval aspects; S * d_k is the packed key width
    d_k: int
    r: int = 0                # low-rank assembly rank (0: value rows only)
    T: float = 1.0
    lambda_sharp: float = 1.0
    use_sigmoid: bool = False

    @property
    def tokens(self) -> int:
        return self.batch * self.seq_len

    @property
    def key_width(self) -> int:
        return self.S * self.d_k

    @property
    def D(self) -> int:
        """Pool row width: [U | V | b] for r > 0, the value rows (d) otherwise."""
        d = self.d_model
        return 2 * d * self.r + d if self.r > 0 else d


# The benchmark LM configurations: pool keys [N, d] with d = S d_k, values [N, d].
SMALL_CHAR = DWALMConfig(vocab=65, d_model=384, n_layers=6, n_heads=6, seq_len=256, batch=16,
                         pool_rows=65536, top_k=32, S=6, d_k=64)
LARGE_1B = DWALMConfig(vocab=32000, d_model=2048, n_layers=24, n_heads=16, seq_len=2048, batch=8,
                       pool_rows=4194304, top_k=64, S=16, d_k=128)
LARGE_7B = DWALMConfig(vocab=32000, d_model=4096, n_layers=32, n_heads=32, seq_len=4096, batch=4,
                       pool_rows=16777216, top_k=128, S=32, d_k=128)
# The reference's own 1B model (configs/large_1b.py:31-70): d_A = d_B = 1280,
# pool 16384 x 21760 ([U | V | b], r = 8), k_max 16, S = 8 aspects of d_k = 64,
# 16 heads, 12 assembly layers, seq 1024 (batch 8), vocab 64400.
REF_1B = DWALMConfig(vocab=64400, d_model=1280, n_layers=12, n_heads=16, seq_len=1024, batch=8,
                     pool_rows=16384, top_k=16, S=8, d_k=64, r=8)

CONFIGS = {"small_char": SMALL_CHAR, "large_1b": LARGE_1B, "large_7b": LARGE_7B,
           "ref_1b": REF_1B}


def _rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """RoPE as bf16 tensor ops: rotate (even, odd) pairs, concatenated like the
    reference (parts.py:17-25).  The forward runs ``lm_ops.rope_qk`` instead, which
    equals this bit for bit."""
    x1, x2 = x[..., ::2], x[..., 1::2]
    return torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)


@dataclass(frozen=True)
class ChunkStep:
    """What the blocks of one ``DWALM.extend`` share: the rows' rotations and cache slots, and
    the sequences they belong to."""

    cache: PagedKVCache
    cos: torch.Tensor          # bf16 [T, dh / 2] by row
    sin: torch.Tensor
    slots: torch.Tensor        # int64 [T]
    block_table: torch.Tensor
    lengths: torch.Tensor
    q_start: torch.Tensor
    max_q: int
    padded: bool               # rows may follow the last sequence's
    tree_mask: torch.Tensor | None = None  # int64 [T, W]: the rows are nodes of trees


def plan_rows(tokens: int) -> int:
    """The row count that a chunk of ``tokens`` rows is planned for: a power of two up to one
    tile of the score kernel (128 rows), whole tiles up to 1024, then eight counts to an
    octave: 63 counts up to 65536 rows, and at most an eighth more rows above 1024."""
    if tokens <= 128:
        return 1 << max(tokens - 1, 0).bit_length()
    step = max(128, 1 << ((tokens - 1).bit_length() - 4))
    return -(-tokens // step) * step


class ChunkPlan:
    """A retrieval plan for chunks of up to its rows: what lies behind a chunk's queries is
    whatever was there before, and dropped."""

    def __init__(self, retriever: Retriever):
        self.retriever = retriever
        with torch.inference_mode(False):  # written in and out of that mode
            self.queries = torch.zeros((retriever.M, retriever.d_k), dtype=torch.bfloat16,
                                       device=retriever.device)
        self._head = (0, None, None)  # a row count, its part of the queries and of the results

    @property
    def keys(self) -> torch.Tensor:
        return self.retriever.keys

    def __call__(self, queries: torch.Tensor, params: torch.Tensor | None = None):
        T = queries.shape[0]
        if T == self.retriever.M:
            return self.retriever(queries, params=params)
        rows, head, results = self._head
        if rows != T:  # the blocks of a forward ask for the same
            with torch.inference_mode(False):
                head = self.queries[:T]
        head.copy_(queries)
        whole = self.retriever(self.queries, params=params)  # the plan's own buffers, always the same
        if rows != T:
            results = tuple(x if x is None else x[:T] for x in whole)
            self._head = (T, head, results)
        return results


def _rope_theta(dh: int, device) -> torch.Tensor:
    return 1.0 / (10000.0 ** (torch.arange(0, dh, 2, device=device) / dh))


class CausalSelfAttention(nn.Module):
    """parts.py:30-83: LayerNorm -> QKV -> RoPE -> causal softmax attention -> proj, residual."""

    def __init__(self, d: int, n_heads: int, seq_len: int, device, dtype):
        super().__init__()
        assert d % n_heads == 0
        self.h, self.dh = n_heads, d // n_heads
        self.norm = nn.LayerNorm(d, device=device, dtype=dtype)
        self.qkv = nn.Linear(d, 3 * d, bias=False, device=device, dtype=dtype)
        self.proj = nn.Linear(d, d, bias=False, device=device, dtype=dtype)
        f = torch.outer(torch.arange(seq_len, device=device, dtype=torch.float32),
                        _rope_theta(self.dh, device))
        self.register_buffer("cos", f.cos().to(dtype), persistent=False)
        self.register_buffer("sin", f.sin().to(dtype), persistent=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, S, C = x.shape
        qkv = self.qkv(self.norm(x))
        # RoPE of q and k in one kernel, bit-identical to _rope on each
        q, k = rope_qk(qkv, self.cos, self.sin, self.h, self.dh)
        v = qkv[..., 2 * C:].view(B, S, self.h, self.dh).transpose(1, 2)
        o = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return x + self.proj(o.transpose(1, 2).reshape(B, S, C))

    def extend(self, x: torch.Tensor, step: ChunkStep, layer: int) -> torch.Tensor:
        """The same for the newest tokens of the sequences in ``step`` (x [1, T, C], packed):
        their keys and values go into the cache, their queries attend to it."""
        _, T, C = x.shape
        qkv = self.qkv(self.norm(x))
        if qkv.dtype != torch.bfloat16 or step.cos.dtype != torch.bfloat16:  # as forward's rope_qk: before pages change
            raise ValueError(f"qkv and cos / sin must be bf16 (got {qkv.dtype} and {step.cos.dtype})")
        q, k, v = (qkv[0, :, i * C:(i + 1) * C].view(T, self.h, self.dh) for i in range(3))
        # rotated as forward's rope_qk does, bit for bit
        q = step.cache.append(layer, q, k, v, step.cos, step.sin, step.slots)
        # the attention leaves a padded batch's last rows as they are
        out = torch.zeros((T, self.h, self.dh), dtype=q.dtype, device=q.device) if step.padded else None
        kw = dict(q_start=step.q_start, max_q=step.max_q, out=out)
        if step.tree_mask is None:
            o = step.cache.attend(layer, q, step.block_table, step.lengths, **kw)
        else:
            o = step.cache.attend_tree(layer, q, step.block_table, step.lengths, step.tree_mask, **kw)
        return x + self.proj(o.view(1, T, C))


class DWABlock(nn.Module):
    """dwa.py:77-130: attention, query_proj, MultiAspectRetrieval (hybrid layout) on
    this repo's kernels, WeightAssembler."""

    def __init__(self, cfg: DWALMConfig, device, dtype, group=None, seed: int = 0):
        super().__init__()
        d = cfg.d_model
        self.cfg = cfg
        self.group = group
        self.attn = CausalSelfAttention(d, cfg.n_heads, cfg.seq_len, device, dtype)
        self.query_proj = nn.Linear(d, d, device=device, dtype=dtype)        # dwa.py:87-96
        self.retrieval = MultiAspectRetrieval(D=cfg.D if cfg.r > 0 else 8, d_A=d, S=cfg.S,
                                              d_k=cfg.d_k, N=cfg.pool_rows, device=device,
                                              dtype=dtype, seed=seed)
        if cfg.r == 0:
            self.retrieval.W_K = None  # the key pool is given (cached packed keys)
        self.assembler = WeightAssembler(d, d, cfg.r, device=device)       # dwa.py:98
        # the retrieval's runtime scalars on the device (tau = w . tau, retrieval.py:168)
        self._params = torch.empty(3, dtype=torch.float32, device=device)

    def queries(self, z: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """([sqrt(w_s) q_s / (|q_s| + 1e-8)]_s packed per position, bf16 [B * seq, S d_k];
        w = softmax(aspect_logits))
        (retrieval.py:159-160 with the aspect weights folded in).  One GEMM for the S
        aspect projections, then one kernel for the normalisation, the packing and
        the retrieval's device scalars (written into ``self._params``)."""
        B, S_len, C = z.shape
        cfg = self.cfg
        W_Q = self.retrieval.W_Q
        q_raw = torch.matmul(z.reshape(B * S_len, C), W_Q.reshape(cfg.S * cfg.d_k, C).t())
        q, w, _ = aspect_queries(q_raw, cfg.S, cfg.d_k, self.retrieval.aspect_logits,
                                 self.retrieval.tau, cfg.lambda_sharp, cfg.T, cfg.use_sigmoid,
                                 params_out=self._params)
        return q, w

    def forward(self, h: torch.Tensor, retriever: Retriever,
                vectors: torch.Tensor | None = None) -> torch.Tensor:
        return self._assemble(self.attn(h), retriever, vectors)

    def extend(self, h: torch.Tensor, plan: ChunkPlan, vectors: torch.Tensor | None,
               step: ChunkStep, layer: int) -> torch.Tensor:
        """``forward`` over the cache: h [1, T, C], the rows of ``step``."""
        return self._assemble(self.attn.extend(h, step, layer), plan, vectors)

    def _assemble(self, h: torch.Tensor, retriever: Retriever | ChunkPlan,
                  vectors: torch.Tensor | None) -> torch.Tensor:
        B, S_len, C = h.shape
        cfg = self.cfg
        z = self.query_proj(h)
        q, w = self.queries(z)  # also the retrieval's {lambda, w . tau, T} in self._params
        if cfg.r > 0:
            # this block's pool keys from the pool vectors (retrieval.py:155-156)
            project_keys_packed(vectors, self.retrieval.W_K, w, out=retriever.keys)
        out, alpha, _, idx = retriever(q, params=self._params)
        hf = h.reshape(B * S_len, C)
        if cfg.r > 0:
            h_mid = self.assembler(hf, alpha, idx, vectors, group=self.group)    # dwa.py:129
        else:
            h_mid = self.assembler.finish(hf, out)                              # b_delta = out
        return h_mid.view(B, S_len, C).to(h.dtype)


class DWALM(nn.Module):
    """dwa.py:133-216 forward: PartA -> DWABlocks over one shared pool -> PartB.

    ``r == 0``: ``pool_keys`` [N_local, S d_k] and ``pool_values`` [N_local, d].
    ``r > 0``: ``pool_values`` are the pool vectors [N_local, D] and ``pool_keys``
    must be None (each block projects its own keys every forward)."""

    def __init__(self, cfg: DWALMConfig, pool_keys: torch.Tensor | None, pool_values: torch.Tensor,
                 group=None, dtype=torch.bfloat16, seed: int = 0):
        super().__init__()
        device = pool_values.device
        torch.manual_seed(seed)
        d = cfg.d_model
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab, d, device=device, dtype=dtype)   # PartA (parts.py:97-98)
        self.embed_proj = nn.Linear(d, d, bias=False, device=device, dtype=dtype)
        self.embed_norm = nn.LayerNorm(d, device=device, dtype=dtype)
        self.blocks = nn.ModuleList(DWABlock(cfg, device, dtype, group, seed=seed * 1000 + i)
                                    for i in range(cfg.n_layers))
        self.head_norm = nn.LayerNorm(d, device=device, dtype=dtype)        # PartB (parts.py:146-176)
        self.fc1 = nn.Linear(d, 4 * d, device=device, dtype=dtype)
        self.fc2 = nn.Linear(4 * d, cfg.vocab, device=device, dtype=dtype)
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, std=math.sqrt(2.0 / m.in_features))
                if m.bias is not None:
                    nn.init.zeros_(m.bias)
        if cfg.r > 0:
            if pool_keys is not None:
                raise ValueError("with r > 0 the blocks project their own keys: pass pool_keys=None")
            self.vectors = pool_values
            values = None
        else:
            if pool_keys is None or pool_keys.shape[1] != cfg.key_width:
                raise ValueError(f"pool_keys must be [N, {cfg.key_width}]")
            self.vectors = None
            # converted once, not by every plan
            pool_keys, values = _as_bf16_rows(pool_keys, "pool_keys"), _check_values(pool_values)

        def plan(tokens: int) -> Retriever:
            # r > 0: a key buffer of the plan's own, rewritten by each block's projection before
            # its retrieval, so that plans may be in use at the same time
            keys = pool_keys if pool_keys is not None else torch.empty(
                (pool_values.shape[0], cfg.key_width), dtype=torch.bfloat16, device=device)
            return Retriever(keys, values, tokens, cfg.top_k, lambda_sharp=cfg.lambda_sharp, T=cfg.T,
                             use_sigmoid=cfg.use_sigmoid, group=group)

        self._plan = plan
        # one retrieval plan shared by all blocks (same pool, same token count)
        self.retriever = plan(cfg.tokens)
        self._chunk_plans: dict[int, ChunkPlan] = {}

    def _chunk_plan(self, tokens: int) -> ChunkPlan:
        """The plan of chunks of ``tokens`` rows; made where there is none."""
        rows = plan_rows(tokens)
        plan = self._chunk_plans.get(rows)
        if plan is None:
            plan = self._chunk_plans[rows] = ChunkPlan(self._plan(rows))
        return plan

    def _retrievers(self) -> list[Retriever]:
        return [self.retriever] + [p.retriever for p in self._chunk_plans.values()]

    def status(self) -> int:
        """The first device status that a retrieval of any call so far left (0: none; waits for the
        device)."""
        torch.cuda.synchronize(self.embed.weight.device)
        return next((s for s in (r.status() for r in self._retrievers()) if s), 0)

    def close(self) -> None:
        """Releases the plans' exchange buffers (collective on a sharded pool: every rank, after its
        last call).  The model is unusable afterwards."""
        for r in self._retrievers():
            r.close()
        self._chunk_plans.clear()

    @torch.no_grad()
    def forward(self, token_ids: torch.Tensor) -> torch.Tensor:
        h = self.embed_norm(self.embed_proj(self.embed(token_ids)))
        for blk in self.blocks:
            h = blk(h, self.retriever, self.vectors)
        return self.fc2(F.gelu(self.fc1(self.head_norm(h))))

    def new_cache(self, n_pages: int, page_size: int = 64,
                  dtype: torch.dtype = torch.bfloat16) -> PagedKVCache:
        """An empty cache for this model (bfloat16, or float8_e4m3fn at half the size)."""
        cfg = self.cfg
        return PagedKVCache(cfg.n_layers, n_pages, page_size, cfg.n_heads, cfg.d_model // cfg.n_heads,
                            dtype=dtype, device=self.embed.weight.device)

    @torch.no_grad()
    def extend(self, token_ids: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor,
               lengths: torch.Tensor, q_start: torch.Tensor | None = None,
               max_q: int | None = None, *, parents: torch.Tensor | None = None) -> torch.Tensor:
        """Logits [T, vocab] of the newest tokens of B sequences, whose earlier tokens are cached.

        ``token_ids`` [T] packs the new tokens: rows q_start[b] to q_start[b + 1] - 1 (int32
        [B + 1]) of sequence b, or T / B rows each without ``q_start``.  ``lengths`` int32 [B]
        counts each sequence's tokens, the new ones with them, and ``block_table`` int32
        [B, max_pages] holds its pages.  ``max_q`` bounds the new tokens of any sequence.
        Rows of no sequence (a padded batch; their tokens are in the vocabulary too) attend to
        nothing.

        With ``parents`` (int32 [T], as ``kv_cache.tree_masks`` takes them) a sequence's new tokens are the
        nodes of a tree: each follows its parent, and sees the tokens cached before the tree, its
        ancestors and itself.  (``max_q`` is 4096 at most then.)

        The retrieval is planned once for all row counts T that ``plan_rows`` rounds to the
        same (a captured graph needs such a call before).  Calls that share a plan share its
        buffers: they, and the graphs that hold them, belong on one stream.  Calls of different
        plans, and ``forward``, may run on different streams at the same time.  On a row-sharded pool every rank calls with
        the same tokens in the same order."""
        T = token_ids.shape[0]
        if token_ids.dim() != 1:
            raise ValueError("token_ids must be [T]")
        B = lengths.shape[0]
        padded = q_start is not None
        if q_start is None:
            if B == 0 or T % B:
                raise ValueError(f"without q_start {T} rows must be equal chunks of {B} sequences")
            q_start = torch.arange(0, T + 1, T // B, dtype=torch.int32, device=token_ids.device) \
                if T else torch.zeros(B + 1, dtype=torch.int32, device=token_ids.device)
            max_q = T // B
        if T == 0:
            return torch.empty((0, self.cfg.vocab), dtype=self.fc2.weight.dtype, device=token_ids.device)
        plan = self._chunk_plan(T)
        slots, positions = cache.slots(block_table, lengths, q_start, T)
        max_q = T if max_q is None else max_q
        mask = None
        if parents is not None:
            mask, depth = tree_masks(parents, q_start=q_start, max_q=max_q, status=cache.status)
            row, start = torch.arange(T, device=q_start.device), q_start.long()
            node = row - start[(torch.searchsorted(start, row, right=True) - 1).clamp(0, B - 1)]
            positions = positions - node + depth  # a node's place in its path, not in the cache
        dh = self.cfg.d_model // self.cfg.n_heads
        f = torch.outer(positions.float(), _rope_theta(dh, positions.device))
        dtype = self.embed.weight.dtype
        step = ChunkStep(cache, f.cos().to(dtype), f.sin().to(dtype), slots, block_table, lengths,
                         q_start, max_q, padded, mask)
        h = self.embed_norm(self.embed_proj(self.embed(token_ids[None])))
        for i, blk in enumerate(self.blocks):
            h = blk.extend(h, plan, self.vectors, step, i)
        return self.fc2(F.gelu(self.fc1(self.head_norm(h))))[0]

    @torch.no_grad()
    def verify(self, last_tokens: torch.Tensor, draft_tokens: torch.Tensor,
               draft_probs: torch.Tensor | None, accept_u: torch.Tensor, sample_u: torch.Tensor,
               cache: PagedKVCache, block_table: torch.Tensor, lengths: torch.Tensor, *,
               temperature: float = 1.0,
               draft_lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """One speculative step: score K drafted tokens of every sequence at once and keep what
        ``verify_drafts`` lets stand.

        ``last_tokens`` int [B] (each sequence's newest token, not yet cached) and ``draft_tokens``
        int32 [B, K] are appended to the ``lengths`` (int32 [B]) cached tokens; the pages in
        ``block_table`` must have room for K + 1 more.  Sequence b has ``draft_lengths[b]``
        drafts (int32 [B], default K each); what follows them may be any number.  Returns (n_accepted int32 [B],
        tokens int32 [B, K + 1] as ``verify_drafts``, new lengths int32 [B]: the cached tokens
        that stay).  tokens[b, n_accepted[b]] is the next step's ``last_tokens[b]``.  A last token
        outside the vocabulary (the -1 of a step without probability mass) is reported in the
        cache's status; its sequence gets no tokens, only -1, and stays as long as it was.
        ``temperature`` divides the logits and is positive (for the best token alone, a small one)."""
        if not isinstance(temperature, torch.Tensor) and not 1e-30 <= temperature <= 1e30:
            raise ValueError(f"temperature must be a positive number, of 1e-30 to 1e30 (got {temperature})")
        if draft_tokens.dim() != 2:
            raise ValueError("draft_tokens must be int32 [B, K]")
        B, K = draft_tokens.shape
        # before the chunk is written: verify_drafts would refuse these after it
        for name, t, dtype, shape in (("draft_tokens", draft_tokens, torch.int32, (B, K)),
                                      ("draft_probs", draft_probs, torch.float32, (B, K, self.cfg.vocab)),
                                      ("accept_u", accept_u, torch.float32, (B, K)),
                                      ("sample_u", sample_u, torch.float32, (B,)),
                                      ("draft_lengths", draft_lengths, torch.int32, (B,))):
            if t is None and name in ("draft_probs", "draft_lengths"):
                continue
            if t is None or t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)}")
        if last_tokens.numel() != B or last_tokens.is_floating_point():
            raise ValueError(f"last_tokens must be integers [{B}]")
        chunk = torch.cat([last_tokens.view(B, 1).to(draft_tokens.dtype), draft_tokens], 1)
        chunk = chunk.clamp(0, self.cfg.vocab - 1)  # a draft outside falls below
        last = last_tokens.view(B)
        lost = (last < 0) | (last >= self.cfg.vocab)
        logits = self.extend(chunk.reshape(-1).long(), cache, block_table, lengths + (K + 1))
        probs = torch.softmax(logits.float().view(B, K + 1, -1) / temperature, -1)
        accepted, tokens = verify_drafts(probs, draft_tokens, draft_probs, accept_u, sample_u,
                                         draft_lengths=draft_lengths)
        cache.report(lost)
        accepted = torch.where(lost, 0, accepted)
        return accepted, torch.where(lost[:, None], -1, tokens), torch.where(lost, lengths, lengths + 1 + accepted)


    @torch.no_grad()
    def verify_tree(self, last_tokens: torch.Tensor, tree_tokens: torch.Tensor, parents: torch.Tensor,
                    sample_u: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor,
                    lengths: torch.Tensor, *,
                    temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """One speculative step with a tree of drafts for every sequence: score them all at once, walk
        down as far as the drawn tokens are drafts, and keep that path in the cache.

        Draft i = 1 .. N of sequence b is ``tree_tokens``[b, i - 1] (int32 [B, N]) and follows draft
        ``parents``[b, i - 1] (int32 [B, N], or [N] for all; below i), or ``last_tokens``[b] (int [B], the sequence's
        newest token, not yet cached) where that is 0; -1 where there is no such draft.  They are appended to the ``lengths`` (int32 [B])
        cached tokens; the pages in ``block_table`` must have room for N + 1 more.  ``sample_u`` f32
        [B, D + 1] are the uniform numbers of the draws, D the most drafts that may stand.  Returns
        (n_accepted int32 [B], tokens int32 [B, D + 1]: the standing drafts, the token drawn after
        them, then -1; new lengths int32 [B]: the cached tokens that stay).  tokens[b, n_accepted[b]] is
        the next step's ``last_tokens[b]``.  A last token outside the vocabulary is reported in the cache's status; its
        sequence gets no tokens, only -1, and stays as long as it was.  ``temperature`` as for ``verify``."""
        if not isinstance(temperature, torch.Tensor) and not 1e-30 <= temperature <= 1e30:
            raise ValueError(f"temperature must be a positive number, of 1e-30 to 1e30 (got {temperature})")
        if tree_tokens.dim() != 2 or tree_tokens.dtype != torch.int32:
            raise ValueError("tree_tokens must be int32 [B, N]")
        B, N = tree_tokens.shape
        if parents.dtype != torch.int32 or tuple(parents.shape) not in ((N,), (B, N)):
            raise ValueError(f"parents must be int32 {[B, N]} or {[N]}")
        if sample_u.dtype != torch.float32 or sample_u.dim() != 2 or sample_u.shape[0] != B \
                or sample_u.shape[1] < 1 or not sample_u.is_contiguous():
            raise ValueError(f"sample_u must be a contiguous torch.float32 [{B}, D + 1]")
        if last_tokens.numel() != B or last_tokens.is_floating_point():
            raise ValueError(f"last_tokens must be integers [{B}]")
        if N + 1 > 4096:
            raise ValueError(f"a tree has 4095 drafts at most (got {N})")
        last = last_tokens.view(B)
        lost = (last < 0) | (last >= self.cfg.vocab)
        chunk = torch.cat([last.view(B, 1).to(torch.int32), tree_tokens], 1).reshape(-1)
        above = torch.cat([torch.full((B, 1), -1, dtype=torch.int32, device=chunk.device),
                           parents.expand(B, N)], 1).reshape(-1)
        logits = self.extend(chunk.clamp(0, self.cfg.vocab - 1).long(), cache, block_table, lengths + (N + 1),
                             parents=above)
        probs = torch.softmax(logits.float() / temperature, -1)
        # a draft outside the vocabulary is never drawn
        accepted, tokens, path = verify_tree(probs, chunk, above, sample_u)
        cache.report(lost)
        cache.keep(block_table, lengths, path, torch.where(lost, -1, accepted))
        accepted = torch.where(lost, 0, accepted)
        return accepted, torch.where(lost[:, None], -1, tokens), torch.where(lost, lengths, lengths + 1 + accepted)


class GraphedForward:
    """The LM forward captured once in a CUDA graph and replayed.

    Every launch of the forward — dense layers, the retrieval kernels of each
    block, their bound resets — goes into one graph, so a small model is not
    bound by per-kernel launch latency.  Capture runs after two eager warm-up
    forwards on a side stream (kernel attributes and tensor maps are set up
    there).  Single-process use only: the graph must not contain collectives.
    """

    def __init__(self, model: DWALM, token_ids: torch.Tensor):
        if model.retriever.world != 1:
            raise ValueError("GraphedForward is for one process; sharded pools use eager forward")
        self.model = model
        self.tokens = token_ids.clone()
        side = torch.cuda.Stream(device=token_ids.device)
        side.wait_stream(torch.cuda.current_stream(token_ids.device))
        with torch.cuda.stream(side):
            for _ in range(2):
                model(self.tokens)
        torch.cuda.current_stream(token_ids.device).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = model(self.tokens)

    def __call__(self, token_ids: torch.Tensor) -> torch.Tensor:
        self.tokens.copy_(token_ids)
        self.graph.replay()
        return self.logits
