"""CPU: the serving operators reject what their kernels cannot take, in Python
before anything reaches the library and at the C ABI before anything is launched
(no GPU is touched)."""
import pytest
import torch

from computd_b200 import _lib
from computd_b200.kv_cache import (kv_cache_read, kv_cache_write, paged_attention, verify_drafts)

FAKE = 0x10000  # 16-byte aligned, never dereferenced: validation fails before any launch


def test_python_calls_refuse_host_tensors():
    c = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache_write(x, x, c, c, slots)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache_read(c, c, slots)
    with pytest.raises(ValueError, match="CUDA"):
        paged_attention(x, c, c, torch.zeros((3, 1), dtype=torch.int32), torch.ones(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        verify_drafts(torch.zeros(1, 2, 8), torch.zeros((1, 1), dtype=torch.int32),
                      torch.zeros(1, 1, 8), torch.zeros(1, 1), torch.zeros(1))


def test_python_calls_refuse_other_objects_and_gradients():
    c = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="torch.Tensor"):
        kv_cache_read([1], c, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="grad"):
        kv_cache_read(c.clone().requires_grad_(), c, torch.zeros(3, dtype=torch.int64))


def test_paged_kv_cache_refuses_bad_sizes():
    from computd_b200 import PagedKVCache

    good = dict(n_layers=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    cache = PagedKVCache(**good, dtype=torch.float8_e4m3fn)
    assert cache.k.shape == (1, 4, 2, 16, 64) and cache.k_scale.shape == (1, 4, 2, 16)
    for kw in (dict(page_size=24), dict(head_dim=72), dict(head_dim=256), dict(n_pages=0),
               dict(dtype=torch.float16)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**good, **kw})
    with pytest.raises(ValueError):
        cache.read(1, torch.zeros(1, dtype=torch.int64))


def test_slots_of_packed_chunks():
    from computd_b200 import PagedKVCache

    cache = PagedKVCache(1, 9, 16, 1, 16)
    table = torch.tensor([[3, 5], [8, 0], [1, 2]], dtype=torch.int32)
    lengths = torch.tensor([18, 3, 40], dtype=torch.int32)  # the last does not fit its pages
    start = torch.tensor([0, 3, 3, 8], dtype=torch.int32)
    slots, positions = cache.slots(table, lengths, start, 10)
    assert positions[:3].tolist() == [15, 16, 17]
    assert slots.tolist() == [3 * 16 + 15, 5 * 16, 5 * 16 + 1] + [-1] * 5 + [-1, -1]
    # more new tokens than the length has: the first have no place
    slots, _ = cache.slots(table, torch.tensor([2, 0, 0], dtype=torch.int32),
                           torch.tensor([0, 4, 4, 4], dtype=torch.int32), 4)
    assert slots.tolist() == [-1, -1, 48, 49]


def cache(**kw):
    a = dict(k_cache=FAKE, v_cache=FAKE, k_scale=None, v_scale=None, H=2, d=64, n_pages=4,
             page_size=16, ld_page=2 * 16 * 64, ld_scale=32)
    a.update({k: v for k, v in kw.items() if k in a})
    return a


BAD_CACHE = [
    (dict(k_cache=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(v_cache=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(k_cache=FAKE + 8), _lib.DWA_ERR_INVALID_ARG),
    (dict(k_scale=FAKE), _lib.DWA_ERR_INVALID_ARG),           # one scale without the other
    (dict(H=0), _lib.DWA_ERR_INVALID_ARG),
    (dict(n_pages=0), _lib.DWA_ERR_INVALID_ARG),
    (dict(n_pages=2 ** 31), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(d=24, ld_page=2 * 16 * 24), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(d=0), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(d=144, ld_page=2 * 16 * 144), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(page_size=48, ld_page=2 * 48 * 64), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(page_size=8), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(ld_page=2 * 16 * 64 - 64), _lib.DWA_ERR_INVALID_ARG),
    (dict(ld_page=2 * 16 * 64 + 8), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(k_scale=FAKE, v_scale=FAKE, ld_scale=31), _lib.DWA_ERR_INVALID_ARG),
]


def write(**kw):
    c = cache(**kw)
    a = dict(k=FAKE, v=FAKE, bf16=1, T=8, kt=128, kh=64, vt=128, vh=64, slots=FAKE)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.load().dwa_kv_write(a["k"], a["v"], a["bf16"], a["T"], c["H"], c["d"], a["kt"], a["kh"],
                                    a["vt"], a["vh"], a["slots"], c["k_cache"], c["v_cache"],
                                    c["k_scale"], c["v_scale"], c["n_pages"], c["page_size"],
                                    c["ld_page"], c["ld_scale"], None, None)


def read(**kw):
    c = cache(**kw)
    a = dict(slots=FAKE, T=8, ko=FAKE, vo=FAKE)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.load().dwa_kv_read(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], a["slots"],
                                   a["T"], c["H"], c["d"], c["n_pages"], c["page_size"], c["ld_page"],
                                   c["ld_scale"], a["ko"], a["vo"], 0, None, None)


def attention(**kw):
    c = cache(**kw)
    a = dict(q=FAKE, T=8, heads=4, q_ld=256, table=FAKE, ld_table=3, max_pages=3, lengths=FAKE,
             q_start=FAKE, B=2, max_q=8, scale=0.125, out=FAKE, out_ld=256, status=None)
    a.update({k: v for k, v in kw.items() if k in a})
    return _lib.load().dwa_paged_attention(
        a["q"], a["T"], a["heads"], c["d"], a["q_ld"], c["k_cache"], c["v_cache"], c["k_scale"],
        c["v_scale"], c["H"], c["n_pages"], c["page_size"], c["ld_page"], c["ld_scale"], a["table"],
        a["ld_table"], a["max_pages"], a["lengths"], a["q_start"], a["B"], a["max_q"], a["scale"],
        a["out"], a["out_ld"], a["status"], None)


@pytest.mark.parametrize("kw,status", BAD_CACHE)
@pytest.mark.parametrize("call", [write, read, attention])
def test_bad_caches(call, kw, status):
    assert call(**kw) == status, _lib.last_error()
    assert _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(k=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(slots=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(k=FAKE + 8), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(kt=132), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(vh=4), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(bf16=0, vh=2), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(kt=-128), _lib.DWA_ERR_INVALID_ARG),
])
def test_bad_writes(kw, status):
    assert write(**kw) == status, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(ko=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(vo=FAKE + 2), _lib.DWA_ERR_INVALID_ARG),
    (dict(T=2 ** 31), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
])
def test_bad_reads(kw, status):
    assert read(**kw) == status, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(B=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(heads=3), _lib.DWA_ERR_UNSUPPORTED_SHAPE),           # not a multiple of H_kv
    (dict(q=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(table=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(q_ld=128), _lib.DWA_ERR_INVALID_ARG),
    (dict(q_ld=260), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(out=FAKE + 4), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(ld_table=2), _lib.DWA_ERR_INVALID_ARG),
    (dict(max_q=0), _lib.DWA_ERR_INVALID_ARG),
    (dict(max_q=2 ** 31 - 1), _lib.DWA_ERR_UNSUPPORTED_SHAPE),  # times two query heads
    (dict(q_start=None, T=9), _lib.DWA_ERR_INVALID_ARG),       # not B equal chunks
    (dict(q_start=None, max_q=3), _lib.DWA_ERR_INVALID_ARG),
    (dict(q_start=None, B=0), _lib.DWA_ERR_INVALID_ARG),       # rows of no sequence
    (dict(scale=3e38), _lib.DWA_ERR_INVALID_ARG),              # log2(e) times it is infinite
    (dict(scale=float("nan")), _lib.DWA_ERR_INVALID_ARG),
    (dict(scale=float("inf")), _lib.DWA_ERR_INVALID_ARG),
    (dict(scale=-1.0), _lib.DWA_ERR_INVALID_ARG),
    (dict(lengths=FAKE + 2), _lib.DWA_ERR_INVALID_ARG),
    (dict(status=FAKE + 1), _lib.DWA_ERR_INVALID_ARG),
    (dict(max_pages=2 ** 28), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
])
def test_bad_attention(kw, status):
    assert attention(**kw) == status, _lib.last_error()


def test_empty_calls_are_noops():
    assert write(T=0, k=None) == 0 and read(T=0, ko=None) == 0
    assert attention(T=0, q=None) == 0 and attention(B=0, lengths=None) == 0
    assert verify(B=0, target=None) == 0


def verify(**kw):
    a = dict(target=FAKE, draft=FAKE, bf16=0, tokens=FAKE, u=FAKE, r=FAKE, lengths=None, B=2, K=3, V=10,
             n=FAKE, out=FAKE)
    a.update(kw)
    return _lib.load().dwa_verify_drafts(a["target"], a["draft"], a["bf16"], a["tokens"], a["u"], a["r"],
                                         a["lengths"], a["B"], a["K"], a["V"], a["n"], a["out"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(K=-1), _lib.DWA_ERR_INVALID_ARG),
    (dict(V=0), _lib.DWA_ERR_INVALID_ARG),
    (dict(target=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(tokens=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(r=None), _lib.DWA_ERR_INVALID_ARG),
    (dict(target=FAKE + 2), _lib.DWA_ERR_INVALID_ARG),
    (dict(lengths=FAKE + 2), _lib.DWA_ERR_INVALID_ARG),
    (dict(V=2 ** 30 + 1), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
    (dict(B=2 ** 30), _lib.DWA_ERR_UNSUPPORTED_SHAPE),
])
def test_bad_verifications(kw, status):
    assert verify(**kw) == status, _lib.last_error()
