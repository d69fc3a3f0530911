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


# The stream and device numbers without the objects that torch.cuda.current_stream makes: a third
# of a short call's time on the host.
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


_entries: dict[str, object] = {}  # C entry points by name, once looked up


def _call(name: str, dev: int, *args) -> None:
    """One C call on device `dev`'s current stream, with that device current."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if dev == _current_device():
        st = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _raw_stream(dev))
    if st:
        _lib.check(st, name)


def _cache_args(k_cache, v_cache, k_scale, v_scale):
    """(device number, H_kv, d, pointers, sizes) of a cache as the C ABI takes them.

    The checks here and below compare whole shapes and strides and format a message only
    when they fail: a decoding step's calls are short."""
    dev, dtype, shape, stride = k_cache.get_device(), k_cache.dtype, k_cache.shape, k_cache.stride()
    if dev < 0:
        raise ValueError("k_cache must live on a CUDA device")
    if len(shape) != 4:
        raise ValueError("k_cache must be [n_pages, H_kv, page_size, d]")
    if (v_cache.dtype is not dtype or v_cache.shape != shape or v_cache.stride() != stride
            or v_cache.get_device() != dev):
        raise ValueError("v_cache must be like k_cache (type, shape, strides, device)")
    n_pages, heads, page, d = shape
    ld_page = stride[0]
    if stride[1:] != (page * d, d, 1) or n_pages == 1:
        ld_page = _strided_page(stride, shape, "a cache's pages must be contiguous inside")
    if dtype is _E4M3:
        if k_scale is None or v_scale is None:
            raise ValueError("a float8_e4m3fn cache needs k_scale and v_scale")
        sshape, sstride = shape[:3], k_scale.stride()
        if (k_scale.dtype is not _F32 or v_scale.dtype is not _F32 or k_scale.shape != sshape
                or v_scale.shape != sshape or v_scale.stride() != sstride
                or k_scale.get_device() != dev or v_scale.get_device() != dev):
            raise ValueError("k_scale and v_scale must be f32 [n_pages, H_kv, page_size] with the same "
                             "strides on the cache's device")
        ld_scale = sstride[0]
        if sstride[1:] != (page, 1) or n_pages == 1:
            ld_scale = _strided_page(sstride, sshape, "the scales of a page must be contiguous")
        return dev, heads, d, (k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                               v_scale.data_ptr()), (n_pages, page, ld_page, ld_scale)
    if dtype is not _BF16:
        raise ValueError("k_cache must be bfloat16 or float8_e4m3fn")
    if k_scale is not None or v_scale is not None:
        raise ValueError("a bfloat16 cache has no scales")
    return dev, heads, d, (k_cache.data_ptr(), v_cache.data_ptr(), None, None), \
        (n_pages, page, ld_page, 0)


def _strided_page(stride, shape, what):
    """The distance between pages where a dimension of size 1 may have any stride."""
    dense = 1
    for size, step in zip(reversed(shape[1:]), reversed(stride[1:])):
        if size > 1 and step != dense:
            raise ValueError(what)
        dense *= size
    return stride[0] if shape[0] > 1 else dense


def _array(x, dtype, shape, dev, name):
    """A contiguous tensor's pointer."""
    if (x.dtype is not dtype or x.shape != shape or x.get_device() != dev or not x.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)} on the same device as the "
                         f"others (got {x.dtype} {list(x.shape)} on {x.device})")
    return x.data_ptr()


def _status(x, dev):
    if x.dtype is not _I32 or x.numel() != 1 or x.get_device() != dev:
        raise ValueError("status must be one int32 on the cache's device")
    return x.data_ptr()


def _rows(x, dtypes, heads, d, dev, name):
    """(T, strides of a token and a head) of [T, heads, d] rows."""
    shape, stride = x.shape, x.stride()
    if (x.dtype not in dtypes or len(shape) != 3 or shape[2] != d or x.get_device() != dev
            or (heads is not None and shape[1] != heads) or stride[2] != 1):
        raise ValueError(f"{name} must be [T, {heads or 'H'}, {d}] of {dtypes}, contiguous along d, on the "
                         f"cache's device (got {x.dtype} {list(shape)}, strides {list(stride)}, on {x.device})")
    # a dimension of size 1 may have any stride
    return shape[0], stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else d


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Write T tokens' keys and values (bf16 or f32 [T, H_kv, d], any token and head
    strides that keep rows 16-byte aligned) into slots ``slots`` (int64 [T]).

    A bf16 cache takes the values rounded; an e4m3 cache takes, per (token, head),
    scale = max(amax / 448, 2^-126) and codes e4m3(x / scale).  A vector with a NaN or
    an infinity reads back as NaN.  Slot -1 skips its token; where a slot is named
    twice the later token stays."""
    dev, heads, d, ptrs, sizes = _cache_args(k_cache, v_cache, k_scale, v_scale)
    T, k_tok, k_head = _rows(k, (_BF16, _F32), heads, d, dev, "k")
    T_v, v_tok, v_head = _rows(v, (k.dtype,), heads, d, dev, "v")
    if T_v != T:
        raise ValueError("k and v must have the same number of tokens")
    _call("dwa_kv_write", dev, k.data_ptr(), v.data_ptr(), 1 if k.dtype is _BF16 else 0, T, heads, d,
          k_tok, k_head, v_tok, v_head, _array(slots, _I64, (T,), dev, "slots"), *ptrs, *sizes,
          None if status is None else _status(status, dev))


def kv_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None,
                  status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of slots ``slots`` (int64 [T]) as bf16 [T, H_kv, d] each.

    With ``out`` (two contiguous tensors) the rows of slot -1 stay as they were; without
    it they are zeros."""
    dev, heads, d, ptrs, sizes = _cache_args(k_cache, v_cache, k_scale, v_scale)
    T = slots.shape[0] if slots.dim() == 1 else 0
    slots_ptr = _array(slots, _I64, (T,), dev, "slots")
    if out is None:
        k, v = k_cache.new_empty((2, T, heads, d), dtype=_BF16).unbind(0)
        k_ptr, v_ptr = k.data_ptr(), v.data_ptr()
    else:
        k, v = out
        k_ptr, v_ptr = (_array(x, _BF16, (T, heads, d), dev, "out") for x in (k, v))
    _call("dwa_kv_read", dev, *ptrs, slots_ptr, T, heads, d, *sizes, k_ptr, v_ptr,
          1 if out is None else 0, None if status is None else _status(status, dev))
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
    dev, h_kv, d, ptrs, sizes = _cache_args(k_cache, v_cache, k_scale, v_scale)
    T, q_ld, q_head = _rows(q, (_BF16,), None, d, dev, "q")
    heads = q.shape[1]
    table_shape = block_table.shape
    if (block_table.dtype is not _I32 or len(table_shape) != 2 or block_table.get_device() != dev
            or (table_shape[1] > 1 and block_table.stride(1) != 1)):
        raise ValueError("block_table must be int32 [B, max_pages], contiguous along its rows, on the "
                         "cache's device")
    B, max_pages = table_shape
    if q_start is None:
        start_ptr = None
        if max_q is None:
            max_q = T // B if B else 0
    else:
        start_ptr = _array(q_start, _I32, (B + 1,), dev, "q_start")
        if max_q is None:
            max_q = T
    if out is None:
        out = q.new_empty((T, heads, d))
        out_ld = heads * d
    else:
        T_out, out_ld, out_head = _rows(out, (_BF16,), heads, d, dev, "out")
        if T_out != T or out_head != d:
            raise ValueError("out must be like q, contiguous over heads and d")
    if q_head != d:
        raise ValueError("q must be contiguous over heads and d")
    _call("dwa_paged_attention", dev, q.data_ptr(), T, heads, d, q_ld or heads * d, *ptrs, h_kv, *sizes,
          block_table.data_ptr(), block_table.stride(0) if B > 1 else max_pages, max_pages,
          _array(lengths, _I32, (B,), dev, "lengths"), start_ptr, B, max_q,
          d ** -0.5 if scale is None else scale, out.data_ptr(), out_ld or heads * d,
          None if status is None else _status(status, dev))
    return out


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
        # DWA_ERR_DEVICE_CHECK once a call met a bad slot, page, length or row range
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

    def read(self, layer: int, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``kv_cache_read`` from one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return kv_cache_read(k_cache, v_cache, slots, **more)

    def attend(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
               **kw) -> torch.Tensor:
        """``paged_attention`` over one layer."""
        k_cache, v_cache, more = self._layer(layer)
        return paged_attention(q, k_cache, v_cache, block_table, lengths, **more, **kw)

    def slots(self, block_table: torch.Tensor, lengths: torch.Tensor, q_start: torch.Tensor,
              n_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(slots int64, positions int64) of the newest tokens of every sequence, row by row of
        a packed chunk of ``n_tokens`` rows: row q_start[b] + i is token lengths[b] - n + i of
        sequence b.  Rows behind q_start[-1], and new tokens that ``lengths`` leaves no
        place for, get slot -1."""
        row = torch.arange(n_tokens, device=q_start.device)
        start, length, table = q_start.long(), lengths.long(), block_table.long()
        seq = (torch.searchsorted(start, row, right=True) - 1).clamp(0, length.shape[0] - 1)
        position = length[seq] - start[seq + 1] + row
        fine = (row < start[-1]) & (position >= 0) & (position < table.shape[1] * self.page_size)
        at = torch.where(fine, position, 0)
        page = table[seq, at // self.page_size]
        return torch.where(fine, page * self.page_size + at % self.page_size, -1), at

    def check(self) -> None:
        """Raise ``DWAError`` if a call so far met a bad slot, page, length or row range (waits
        for the device)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise _lib.DWAError(code, "PagedKVCache", "a slot, page number, length or row range was "
                                "outside the cache or the call")


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
    dev, dtype, shape = target_probs.get_device(), target_probs.dtype, target_probs.shape
    if dev < 0:
        raise ValueError("target_probs must live on a CUDA device")
    if dtype not in (_F32, _BF16) or len(shape) != 3 or shape[1] < 1 or not target_probs.is_contiguous():
        raise ValueError("target_probs must be a contiguous float32 or bfloat16 [B, K + 1, V]")
    B, K1, V = shape
    K = K1 - 1
    accepted = draft_tokens.new_empty((B,), dtype=_I32)
    tokens = draft_tokens.new_empty((B, K1), dtype=_I32)
    _call("dwa_verify_drafts", dev, target_probs.data_ptr(),
          None if draft_probs is None else _array(draft_probs, dtype, (B, K, V), dev, "draft_probs"),
          1 if dtype is _BF16 else 0, _array(draft_tokens, _I32, (B, K), dev, "draft_tokens"),
          _array(accept_u, _F32, (B, K), dev, "accept_u"),
          _array(sample_u, _F32, (B,), dev, "sample_u"),
          None if draft_lengths is None else _array(draft_lengths, _I32, (B,), dev, "draft_lengths"),
          B, K, V, accepted.data_ptr(), tokens.data_ptr())
    return accepted, tokens
