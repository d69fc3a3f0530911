"""Serving: the paged key/value cache, attention of new tokens over it, and the
verification of drafted tokens (include/dwa_decode.h).

The reference generates by whole forwards over a growing window
(src/training/trainer.py:258-338); it has no cache.  These are the operators of
a chunk forward over one (``DWALM.extend``, ``DWALM.verify``):

* ``kv_cache_write`` puts new tokens' keys and values into pages, as bf16 or as
  e4m3 with one f32 scale per (token, head); ``kv_cache_read`` brings them back.
* ``paged_attention`` attends from every sequence's newest tokens (one, a few
  drafted ones, a prompt's piece) to its pages.
* ``verify_drafts`` holds drafted tokens against the target's probabilities.
* ``kv_cache_append`` is ``kv_cache_write`` with the rotary embedding of the keys, and the
  queries', on the way.
* ``tree_masks``, ``paged_tree_attention``, ``verify_tree`` and ``kv_cache_keep`` do for a tree of drafted
  tokens (several candidates to a place) what a chunk's causal attention and ``verify_drafts`` do for
  one row of them (``DWALM.verify_tree``).

A tree is a sequence's n newest tokens: node 0 the newest that stands, the others drafts, parents before
children.  The cache holds node j as token length - n + j until ``kv_cache_keep`` moves the path that
stood.

A cache is a pair of tensors [n_pages, H_kv, page_size, d] (bf16, or
float8_e4m3fn with f32 scales [n_pages, H_kv, page_size]); pages may be strided,
what is inside a page is contiguous.  Slot s is token s % page_size of page
s // page_size.  Every call is asynchronous on the current stream, allocates
nothing but its outputs, never waits for the device and can be captured in a
CUDA graph; none has gradients.  Values that only the device sees (slots, page numbers, lengths) are
checked there: a bad one leads to no access but to NaN rows (or a skipped write),
and to ``DWA_ERR_DEVICE_CHECK`` in ``status``, an int32 device word, when given.  (Rows
that a bad row range leaves to no sequence stay as they were.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_BF16, _E4M3, _F32, _I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32


_host_module = None


def _host():
    """The extension module with the checks and the C calls (csrc/host/serving.cpp), bound to the
    loaded library: checked in Python, a decoding step's calls take the host two to three
    times as long as the device."""
    global _host_module
    if _host_module is None:
        lib = _lib.load()
        try:
            from . import _serving as host
        except ImportError as e:
            raise ImportError("computd_b200/_serving.so is missing or does not fit this torch; build it "
                              "with `python -m computd_b200.build`. There is no fallback implementation."
                              ) from e
        host.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                    for name in ("dwa_kv_write", "dwa_kv_read", "dwa_paged_attention",
                                 "dwa_verify_drafts", "dwa_kv_append", "dwa_kv_keep",
                                 "dwa_paged_tree_attention", "dwa_paged_tree_attention_workspace",
                                 "dwa_tree_masks", "dwa_verify_tree")),
                  _lib.check)
        _host_module = host
    return _host_module


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Write T tokens' keys and values (bf16 or f32 [T, H_kv, d], any token and head
    strides that keep rows 16-byte aligned) into slots ``slots`` (int64 [T]).

    A bf16 cache takes the values rounded; an e4m3 cache takes, per (token, head),
    scale = max(amax / 448, 2^-126) and codes e4m3(x / scale).  A vector with a NaN or
    an infinity reads back as NaN.  Slot -1 skips its token; where a slot is named
    twice the later token stays."""
    (_host_module or _host()).kv_write(k, v, k_cache, v_cache, slots, k_scale, v_scale, status)


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None,
                  status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of slots ``slots`` (int64 [T]) as bf16 [T, H_kv, d] each.

    With ``out`` (two contiguous tensors) the rows of slot -1 stay as they were; without
    it they are zeros, and the two results are parts of one allocation: keeping (or saving)
    one keeps both, unless it is cloned."""
    return (_host_module or _host()).kv_read(k_cache, v_cache, slots, k_scale, v_scale, out, status)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, lengths: torch.Tensor, *,
                    q_start: torch.Tensor | None = None, max_q: int | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every sequence's newest tokens over its cached ones (bf16 [T, H, d]).

    ``q`` bf16 [T, H, d] packs the new tokens of B sequences: rows q_start[b] to
    q_start[b + 1] - 1 (int32 [B + 1]), or T / B rows each without ``q_start``.
    ``lengths`` int32 [B] counts the cached tokens, the new ones (written already)
    with them; ``block_table`` int32 [B, max_pages] holds their pages in order.  New
    token i of n attends to the first length - n + i + 1 tokens, query head h to
    key/value head h // (H / H_kv); ``scale`` defaults to d ** -0.5.  A row that sees
    nothing is zeros; rows of no sequence (before q_start[0], from q_start[B] on) are left as
    they were in ``out``, and without it hold anything.

    ``max_q`` bounds the new tokens of any one sequence (default: T); the host picks
    the kernel by it, so a close bound is faster.  A sequence with more gets NaN.  Up to 16
    rows per key/value head (max_q H / H_kv) the probabilities over a bf16 cache keep 16 bits,
    beyond that 8 (over an e4m3 cache 11 either way), as include/dwa_decode.h says.

    What a row may not see does not reach it, NaN and infinities included.  (A new
    token's value that is not finite makes the rows that do see it not finite in its
    channel; an infinity may become NaN there.)"""
    return (_host_module or _host()).attend(q, k_cache, v_cache, block_table, lengths, q_start, max_q,
                                            k_scale, v_scale, scale, out, status)


def kv_cache_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                    positions: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                    status: torch.Tensor | None = None) -> torch.Tensor | None:
    """``kv_cache_write`` of T tokens whose keys are rotated for their positions on the way;
    returns their queries rotated (bf16 [T, H, d]), or None without ``q``.

    ``q`` [T, H, d], ``k`` and ``v`` [T, H_kv, d] (all bf16 or all f32; token and head strides as for
    ``kv_cache_write``), ``cos`` and ``sin`` [n_positions, d / 2] (both bf16 or both f32), ``positions``
    int64 [T] their rows (default: token t has row t).  With x1 = x[0::2] and x2 = x[1::2] a rotated vector is
    [x1 cos - x2 sin, x1 sin + x2 cos].  bf16 tensors with bf16 tables round every step to bf16,
    which equals ``lm_ops.rope_qk`` and ``kv_cache_write`` bit for bit; otherwise all is f32 and rounded once
    (e4m3 keys are coded from their f32 values).  A position outside the tables makes its query
    and keys NaN, and is reported."""
    return (_host_module or _host()).kv_append(q, k, v, cos, sin, k_cache, v_cache, slots, positions, k_scale,
                                               v_scale, q_out, status)


def tree_masks(parents: torch.Tensor, *, q_start: torch.Tensor | None = None, n_trees: int | None = None,
               max_q: int | None = None,
               status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """What the nodes of trees see: (mask int64 [T, W], depth int32 [T]).

    ``parents`` int32 [T] packs the trees' nodes, rows q_start[b] to q_start[b + 1] - 1 (int32
    [B + 1]) of tree b, or ``n_trees`` equal trees (default one): the number of a node's parent in its
    tree, which is below its own, or -1.  Bit j % 64 of word j // 64 of a node's row says that it is node j or
    below it; its depth is the number of nodes above it.  W = ceil(max_q / 64) words, where ``max_q``
    (default: T, or T / n_trees; 4096 at most) bounds a tree's nodes.  A parent that does not come before its node is reported
    and counts as none; rows of no tree (those too
    that only a bad range of rows covers, which is reported), and of one with more than ``max_q`` nodes, are zeros."""
    return (_host_module or _host()).masks(parents, q_start, n_trees, max_q, status)


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         block_table: torch.Tensor, lengths: torch.Tensor, tree_mask: torch.Tensor, *,
                         q_start: torch.Tensor | None = None, max_q: int | None = None,
                         k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                         scale: float | None = None, out: torch.Tensor | None = None,
                         status: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` of new tokens that are the nodes of trees (bf16 [T, H, d]).

    Node i of a sequence's n new tokens attends to its first length - n tokens, and to node j (cached
    as token length - n + j) where bit j % 64 of word j // 64 of its row of ``tree_mask`` (int64 [T, W])
    is set: those of ``tree_masks``, or any others.  Bits from n on count for nothing; a node sees
    itself only if its own bit is set, and one that sees nothing gets zeros.  ``max_q`` bounds a tree's
    nodes, is 64 W at most, and picks the kernel with the sizes of ``q`` and ``block_table``: up to 32
    rows per key/value head, and 64 where tables are narrow, the probabilities over a bf16 cache keep 16
    bits, beyond that 8 (over an e4m3 cache 11 either way), as include/dwa_decode.h says.  Everything else, the other arguments, rows of no sequence and values that are not
    finite, is as there."""
    return (_host_module or _host()).attend_tree(q, k_cache, v_cache, block_table, lengths, q_start, max_q,
                                                 k_scale, v_scale, scale, out, status, tree_mask)


def verify_tree(target_probs: torch.Tensor, tree_tokens: torch.Tensor, parents: torch.Tensor,
                sample_u: torch.Tensor, *,
                q_start: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The walk through verified trees.

    ``target_probs`` [T, V] (f32 or bf16, contiguous) are the target's probabilities behind every node,
    ``tree_tokens`` int32 [T] the nodes' tokens (node 0's is not looked at), ``parents`` int32 [T] as for
    ``tree_masks``, ``sample_u`` f32 [B, steps] uniform in [0, 1); rows q_start[b] to q_start[b + 1] - 1
    (int32 [B + 1]) are tree b, or T / B each.  From node 0 on, step s draws a token from the node's row (the lowest
    index whose running sum exceeds sample_u[b, s] times the row's sum) and goes to the node's first
    child with that token, or ends.  The tokens are distributed as the target's, whatever proposed
    the drafts.  At most steps - 1 drafts are passed.

    Returns (n_accepted int32 [B], tokens int32 [B, steps]: the passed drafts, the last drawn token,
    then -1; path int32 [B, steps]: the nodes passed, 0 first, then -1), parts of one allocation."""
    return (_host_module or _host()).verify_tree(target_probs, tree_tokens, parents, sample_u, q_start)


def kv_cache_keep(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor,
                  path: torch.Tensor, n_accepted: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Move the cached tokens of the paths that stood to where their sequences' tokens belong.

    Sequence b's token start[b] + path[b, i] becomes token start[b] + i for i = 0 .. n_accepted[b]
    (``start`` and ``n_accepted`` int32 [B], ``path`` int32 [B, steps], as ``verify_tree`` returns them), on the
    pages of ``block_table`` (int32 [B, max_pages]).  The caches are one layer's, or all layers'
    [layers, n_pages, H_kv, page_size, d].  Paths ascend from 0 or more; one that does not, or that leaves
    the pages, is reported and its sequence stays as it was."""
    (_host_module or _host()).kv_keep(k_cache, v_cache, block_table, start, path, n_accepted, k_scale, v_scale,
                                      status)


class PagedKVCache:
    """The keys and values of a model's layers on one set of pages.

    ``n_pages`` pages of ``page_size`` (16, 32, 64 or 128) tokens in each of
    ``n_layers`` layers, ``n_kv_heads`` heads of ``head_dim`` (a multiple of 16 up to
    128), bfloat16 or float8_e4m3fn.  A page number means the same tokens in every
    layer, so one block table serves them all; which pages belong to which sequence is
    the caller's.  The methods are this module's calls on one layer."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = _BF16, device=None):
        if dtype not in (_BF16, _E4M3):
            raise ValueError("dtype must be bfloat16 or float8_e4m3fn")
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128")
        if head_dim % 16 or not 16 <= head_dim <= 128:
            raise ValueError("head_dim must be a multiple of 16 up to 128")
        if min(n_layers, n_pages, n_kv_heads) < 1:
            raise ValueError("n_layers, n_pages and n_kv_heads must be positive")
        self.n_layers, self.n_pages, self.page_size = int(n_layers), int(n_pages), int(page_size)
        shape = (self.n_layers, self.n_pages, int(n_kv_heads), self.page_size, int(head_dim))
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = None
        if dtype is _E4M3:
            self.k_scale, self.v_scale = (torch.empty(shape[:4], dtype=_F32, device=device)
                                          for _ in range(2))
        # DWA_ERR_DEVICE_CHECK once a call met a bad slot, page, length, row range or last token
        with torch.inference_mode(False):  # written in and out of that mode
            self.status = torch.zeros((), dtype=_I32, device=device)

    def _layer(self, layer: int):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        if self.k_scale is None:
            return self.k[layer], self.v[layer], {"status": self.status}
        return self.k[layer], self.v[layer], {"k_scale": self.k_scale[layer],
                                              "v_scale": self.v_scale[layer], "status": self.status}

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """``kv_cache_write`` into one layer."""
        k_cache, v_cache, more = self._layer(layer)
        kv_cache_write(k, v, k_cache, v_cache, slots, **more)

    def append(self, layer: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
               sin: torch.Tensor, slots: torch.Tensor, **kw) -> torch.Tensor | None:
        """``kv_cache_append`` to one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return kv_cache_append(q, k, v, cos, sin, k_cache, v_cache, slots, **more, **kw)

    def read(self, layer: int, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``kv_cache_read`` from one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return kv_cache_read(k_cache, v_cache, slots, **more)

    def attend(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
               **kw) -> torch.Tensor:
        """``paged_attention`` over one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return paged_attention(q, k_cache, v_cache, block_table, lengths, **more, **kw)

    def attend_tree(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                    tree_mask: torch.Tensor, **kw) -> torch.Tensor:
        """``paged_tree_attention`` over one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return paged_tree_attention(q, k_cache, v_cache, block_table, lengths, tree_mask, **more, **kw)

    def keep(self, block_table: torch.Tensor, start: torch.Tensor, path: torch.Tensor,
             n_accepted: torch.Tensor) -> None:
        """``kv_cache_keep`` in every layer, in one launch."""
        kv_cache_keep(self.k, self.v, block_table, start, path, n_accepted, k_scale=self.k_scale,
                      v_scale=self.v_scale, status=self.status)

    def slots(self, block_table: torch.Tensor, lengths: torch.Tensor, q_start: torch.Tensor,
              n_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(slots int64, positions int64) of the newest tokens of every sequence, row by row of
        a packed chunk of ``n_tokens`` rows: row q_start[b] + i is token lengths[b] - n + i of
        sequence b.  Rows of no sequence, and new tokens that ``lengths`` leaves no place
        for, get slot -1; tokens on a negative page get -2, which the calls report."""
        row = torch.arange(n_tokens, device=q_start.device)
        start, length, table = q_start.long(), lengths.long(), block_table.long()
        seq = (torch.searchsorted(start, row, right=True) - 1).clamp(0, length.shape[0] - 1)
        position = length[seq] - start[seq + 1] + row
        fine = ((row >= start[seq]) & (row < start[seq + 1]) & (position >= 0)
                & (position < table.shape[1] * self.page_size))
        at = torch.where(fine, position, 0)
        page = table[seq, at // self.page_size]
        slot = torch.where(page < 0, -2, page * self.page_size + at % self.page_size)
        return torch.where(fine, slot, -1), at

    def report(self, bad: torch.Tensor) -> None:
        """Note in ``status`` that ``bad`` (bool, any shape) has a true value, if it has; by an atomic
        maximum, as calls on other streams may note something at the same time."""
        codes = torch.where(bad.flatten(), _lib.DWA_ERR_DEVICE_CHECK, 0).to(_I32)
        self.status.view(1).scatter_reduce_(0, torch.zeros_like(codes, dtype=torch.int64), codes, "amax")

    def check(self) -> None:
        """Raise ``DWAError`` if a call so far met a bad slot, page, length, row range or last
        token (waits for the device)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise _lib.DWAError(code, "PagedKVCache", "a slot, page number, length, row range or last "
                                "token was outside the cache, the call or the vocabulary")


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor,
                  draft_probs: torch.Tensor | None, accept_u: torch.Tensor, sample_u: torch.Tensor, *,
                  draft_lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Hold drafted tokens against the target's probabilities.

    ``target_probs`` [B, K + 1, V] and ``draft_probs`` [B, K, V] (f32 or bf16, contiguous;
    None: the drafter's token had probability 1), ``draft_tokens`` int32 [B, K],
    ``accept_u`` f32 [B, K] and ``sample_u`` f32 [B] uniform in [0, 1), ``draft_lengths``
    int32 [B] (default K each).  Draft i stands while accept_u q(x) < p(x); the first
    that falls is replaced by a draw (by ``sample_u``, the lowest index whose running
    sum exceeds it) from max(p - q, 0), or all stand and a token drawn from the next p
    follows, so that the tokens are distributed as the target's.

    Returns (n_accepted int32 [B], tokens int32 [B, K + 1]: the standing drafts, the drawn
    token, then -1), two parts of one allocation."""
    return (_host_module or _host()).verify(target_probs, draft_tokens, draft_probs, accept_u, sample_u,
                                            draft_lengths)
