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

A cache is a pair of tensors [n_pages, H_kv, page_size, d] (bf16, or
float8_e4m3fn with f32 scales [n_pages, H_kv, page_size]); pages may be strided,
what is inside a page is contiguous.  Slot s is token s % page_size of page
s // page_size.  Every call is asynchronous on the current stream, allocates
nothing but its outputs, never waits for the device and can be captured in a
CUDA graph.  Values that only the device sees (slots, page numbers, lengths) are
checked there: a bad one leads to no access but to NaN rows (or a skipped write),
and to ``DWA_ERR_DEVICE_CHECK`` in ``status``, an int32 device word, when given.
"""
from __future__ import annotations

import torch

from . import _lib

_BF16, _E4M3, _F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32
_I32, _I64 = torch.int32, torch.int64


def _call(fn: str, device: torch.device, *args) -> None:
    """One C call on `device`'s current stream, with that device current."""
    lib = _lib.load()
    index = device.index
    if index == torch.cuda.current_device():
        st = getattr(lib, fn)(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            st = getattr(lib, fn)(*args, torch.cuda.current_stream(device).cuda_stream)
    if st:
        _lib.check(st, fn)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _cache_args(k_cache, v_cache, k_scale, v_scale):
    """(device, pointers and sizes of a cache as the C ABI takes them)."""
    _need(k_cache.is_cuda, "k_cache must live on a CUDA device")
    dtype, shape = k_cache.dtype, k_cache.shape
    _need(dtype in (_BF16, _E4M3), "k_cache must be bfloat16 or float8_e4m3fn")
    _need(len(shape) == 4, "k_cache must be [n_pages, H_kv, page_size, d]")
    dev, stride = k_cache.device, k_cache.stride()
    _need(v_cache.dtype == dtype and v_cache.shape == shape and v_cache.stride() == stride
          and v_cache.device == dev, "v_cache must be like k_cache (type, shape, strides, device)")
    n_pages, heads, page, d = shape
    _need((d == 1 or stride[3] == 1) and (page == 1 or stride[2] == d)
          and (heads == 1 or stride[1] == page * d), "a cache's pages must be contiguous inside")
    ld_page = stride[0] if n_pages > 1 else heads * page * d
    if dtype is _BF16:
        _need(k_scale is None and v_scale is None, "a bfloat16 cache has no scales")
        return dev, (k_cache.data_ptr(), v_cache.data_ptr(), None, None), \
            (n_pages, page, ld_page, 0), heads, d
    _need(k_scale is not None and v_scale is not None, "a float8_e4m3fn cache needs k_scale and v_scale")
    sstride = k_scale.stride()
    for s in (k_scale, v_scale):
        _need(s.dtype == _F32 and s.shape == shape[:3] and s.device == dev and s.stride() == sstride,
              "k_scale and v_scale must be f32 [n_pages, H_kv, page_size] with the same strides on "
              "the cache's device")
    _need((page == 1 or sstride[2] == 1) and (heads == 1 or sstride[1] == page),
          "the scales of a page must be contiguous")
    return dev, (k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()), \
        (n_pages, page, ld_page, sstride[0] if n_pages > 1 else heads * page), heads, d


def _int_arg(x, dtype, dim, dev, name):
    _need(x.dtype == dtype and x.dim() == dim and x.device == dev
          and (dim == 0 or x.shape[-1] <= 1 or x.stride(-1) == 1),
          f"{name} must be a {dim}-D {dtype} tensor on the cache's device, contiguous along its last "
          "dimension")
    return x.data_ptr()


def _status_arg(status, dev):
    if status is None:
        return None
    _need(status.dtype == _I32 and status.numel() == 1 and status.device == dev,
          "status must be one int32 on the cache's device")
    return status.data_ptr()


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Write T tokens' keys and values (bf16 or f32 [T, H_kv, d], any token and head
    strides that keep rows 16-byte aligned) into slots ``slots`` (int64 [T]).

    A bf16 cache takes the values rounded; an e4m3 cache takes, per (token, head),
    scale = max(amax / 448, 2^-126) and codes e4m3(x / scale).  A vector with a NaN or
    an infinity reads back as NaN.  Slot -1 skips its token; where a slot is named
    twice the later token stays."""
    dev, ptrs, sizes, heads, d = _cache_args(k_cache, v_cache, k_scale, v_scale)
    shape = k.shape
    _need(k.dtype in (_BF16, _F32) and v.dtype == k.dtype, "k and v must both be bfloat16 or float32")
    _need(len(shape) == 3 and shape[1] == heads and shape[2] == d and v.shape == shape,
          f"k and v must be [T, {heads}, {d}]")
    _need(k.device == dev and v.device == dev, "k and v must live on the cache's device")
    ks, vs = k.stride(), v.stride()
    _need(ks[2] == 1 and vs[2] == 1, "k and v must be contiguous along d")
    T = shape[0]
    slots_ptr = _int_arg(slots, _I64, 1, dev, "slots")
    _need(slots.shape[0] == T, f"slots must have {T} entries")
    _call("dwa_kv_write", dev, k.data_ptr(), v.data_ptr(), 1 if k.dtype is _BF16 else 0, T, heads, d,
          ks[0] if T > 1 else 0, ks[1] if heads > 1 else 0, vs[0] if T > 1 else 0,
          vs[1] if heads > 1 else 0, slots_ptr, *ptrs, *sizes, _status_arg(status, dev))


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None,
                  status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of slots ``slots`` (int64 [T]) as bf16 [T, H_kv, d] each.

    With ``out`` (two contiguous tensors) the rows of slot -1 stay as they were; without
    it they are zeros."""
    dev, ptrs, sizes, heads, d = _cache_args(k_cache, v_cache, k_scale, v_scale)
    slots_ptr = _int_arg(slots, _I64, 1, dev, "slots")
    shape = (slots.shape[0], heads, d)
    if out is None:
        k, v = (torch.empty(shape, dtype=_BF16, device=dev) for _ in range(2))
        clear = 1
    else:
        k, v = out
        clear = 0
        for x in (k, v):
            _need(x.dtype == _BF16 and x.shape == shape and x.is_contiguous() and x.device == dev,
                  f"out must be two contiguous bfloat16 {list(shape)} on the cache's device")
    _call("dwa_kv_read", dev, *ptrs, slots_ptr, shape[0], heads, d, *sizes, k.data_ptr(),
          v.data_ptr(), clear, _status_arg(status, dev))
    return k, v


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
    nothing is zeros; rows from q_start[B] on are left as they were (in ``out``).

    ``max_q`` bounds the new tokens of any one sequence (default: T); the host picks
    the kernel by it, so a close bound is faster.  A sequence with more gets NaN.

    What a row may not see does not reach it, NaN and infinities included.  (A new
    token's value that is not finite makes the rows that do see it not finite in its
    channel; an infinity may become NaN there.)"""
    dev, ptrs, sizes, h_kv, d = _cache_args(k_cache, v_cache, k_scale, v_scale)
    shape = q.shape
    _need(q.dtype == _BF16 and len(shape) == 3 and shape[2] == d and q.device == dev,
          f"q must be a bfloat16 [T, H, {d}] on the cache's device")
    T, heads, _ = shape
    qs = q.stride()
    _need(qs[2] == 1 and (heads <= 1 or qs[1] == d), "q must be contiguous over heads and d")
    q_ld = qs[0] if T > 1 else heads * d
    table_ptr = _int_arg(block_table, _I32, 2, dev, "block_table")
    lengths_ptr = _int_arg(lengths, _I32, 1, dev, "lengths")
    B, max_pages = block_table.shape
    _need(lengths.shape[0] == B, f"lengths must have {B} entries")
    start_ptr = None
    if q_start is not None:
        start_ptr = _int_arg(q_start, _I32, 1, dev, "q_start")
        _need(q_start.shape[0] == B + 1, f"q_start must have {B + 1} entries")
        if max_q is None:
            max_q = T
    elif max_q is None:
        max_q = T // B if B else 0
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=dev)
        out_ld = heads * d
    else:
        _need(out.dtype == _BF16 and out.shape == shape and out.device == dev,
              f"out must be a bfloat16 {list(shape)} on the cache's device")
        os = out.stride()
        _need(os[2] == 1 and (heads <= 1 or os[1] == d), "out must be contiguous over heads and d")
        out_ld = os[0] if T > 1 else heads * d
    _call("dwa_paged_attention", dev, q.data_ptr(), T, heads, d, q_ld, *ptrs, h_kv, *sizes, table_ptr,
          block_table.stride(0) if B > 1 else max_pages, max_pages, lengths_ptr, start_ptr, B,
          int(max_q), d ** -0.5 if scale is None else float(scale), out.data_ptr(), out_ld,
          _status_arg(status, dev))
    return out


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
    token, then -1)."""
    _need(target_probs.is_cuda, "target_probs must live on a CUDA device")
    dev, dtype = target_probs.device, target_probs.dtype
    _need(dtype in (_F32, _BF16) and target_probs.dim() == 3 and target_probs.is_contiguous(),
          "target_probs must be a contiguous float32 or bfloat16 [B, K + 1, V]")
    B, K1, V = target_probs.shape
    K = K1 - 1
    _need(K >= 0, "target_probs must have at least one position")
    draft_ptr = None
    if draft_probs is not None:
        _need(draft_probs.dtype == dtype and draft_probs.shape == (B, K, V)
              and draft_probs.is_contiguous() and draft_probs.device == dev,
              f"draft_probs must be a contiguous {dtype} [{B}, {K}, {V}] on target_probs' device")
        draft_ptr = draft_probs.data_ptr()
    for x, want, shape, name in ((draft_tokens, _I32, (B, K), "draft_tokens"),
                                 (accept_u, _F32, (B, K), "accept_u"),
                                 (sample_u, _F32, (B,), "sample_u")):
        _need(x.dtype == want and x.shape == shape and x.is_contiguous() and x.device == dev,
              f"{name} must be a contiguous {want} {list(shape)} on target_probs' device")
    lengths_ptr = None
    if draft_lengths is not None:
        _need(draft_lengths.dtype == _I32 and draft_lengths.shape == (B,)
              and draft_lengths.is_contiguous() and draft_lengths.device == dev,
              f"draft_lengths must be a contiguous int32 [{B}] on target_probs' device")
        lengths_ptr = draft_lengths.data_ptr()
    accepted = torch.empty((B,), dtype=_I32, device=dev)
    tokens = torch.empty((B, K1), dtype=_I32, device=dev)
    _call("dwa_verify_drafts", dev, target_probs.data_ptr(), draft_ptr, 1 if dtype is _BF16 else 0,
          draft_tokens.data_ptr(), accept_u.data_ptr(), sample_u.data_ptr(), lengths_ptr, B, K, V,
          accepted.data_ptr(), tokens.data_ptr())
    return accepted, tokens
