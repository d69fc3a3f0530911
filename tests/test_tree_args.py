"""CPU: the operators of draft trees refuse what their kernels cannot take, in Python before anything
reaches the library and at the C ABI before anything is launched (no GPU is touched)."""
import pytest
import torch
from test_decode_args import BAD_CACHE, FAKE, cache

from computd_b200 import _lib
from computd_b200.kv_cache import (kv_cache_append, kv_cache_keep, paged_tree_attention, tree_masks,
                                   verify_tree)

BAD, SHAPE = _lib.DWA_ERR_INVALID_ARG, _lib.DWA_ERR_UNSUPPORTED_SHAPE


def _with(a, kw):
    a.update({k: v for k, v in kw.items() if k in a})
    return a


def append(**kw):
    c = cache(**kw)
    a = _with(dict(q=FAKE, k=FAKE, v=FAKE, bf16=1, T=8, heads=4, qt=256, qh=64, kt=128, kh=64, vt=128, vh=64,
                   cos=FAKE, sin=FAKE, tables_bf16=0, ld_table=32, n_positions=100, positions=FAKE,
                   slots=FAKE, q_out=FAKE, status=None), kw)
    return _lib.load().dwa_kv_append(
        a["q"], a["k"], a["v"], a["bf16"], a["T"], a["heads"], c["H"], c["d"], a["qt"], a["qh"], a["kt"], a["kh"],
        a["vt"], a["vh"], a["cos"], a["sin"], a["tables_bf16"], a["ld_table"], a["n_positions"], a["positions"],
        a["slots"], c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["n_pages"], c["page_size"],
        c["ld_page"], c["ld_scale"], a["q_out"], a["status"], None)


def attention(**kw):
    c = cache(**kw)
    a = _with(dict(q=FAKE, T=8, heads=4, q_ld=256, table=FAKE, ld_table=3, max_pages=3, lengths=FAKE, q_start=FAKE,
                   B=2, max_q=8, mask=FAKE, words=1, scale=0.125, out=FAKE, out_ld=256, status=None), kw)
    return _lib.load().dwa_paged_tree_attention(
        a["q"], a["T"], a["heads"], c["d"], a["q_ld"], c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["H"],
        c["n_pages"], c["page_size"], c["ld_page"], c["ld_scale"], a["table"], a["ld_table"], a["max_pages"],
        a["lengths"], a["q_start"], a["B"], a["max_q"], a["mask"], a["words"], a["scale"], a["out"], a["out_ld"],
        None, 0, a["status"], None)


def keep(**kw):
    c = cache(**kw)
    a = _with(dict(layers=2, ld_layer=4 * 2 * 16 * 64, ld_scale_layer=128, table=FAKE, ld_table=3, max_pages=3,
                   start=FAKE, path=FAKE, kept=FAKE, B=2, steps=4, status=None), kw)
    return _lib.load().dwa_kv_keep(
        c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], a["layers"], a["ld_layer"], a["ld_scale_layer"],
        c["H"], c["d"], c["n_pages"], c["page_size"], c["ld_page"], c["ld_scale"], a["table"], a["ld_table"],
        a["max_pages"], a["start"], a["path"], a["kept"], a["B"], a["steps"], a["status"], None)


def masks(**kw):
    a = _with(dict(parents=FAKE, q_start=FAKE, T=8, B=2, max_q=8, mask=FAKE, words=1, depth=FAKE, status=None), kw)
    return _lib.load().dwa_tree_masks(a["parents"], a["q_start"], a["T"], a["B"], a["max_q"], a["mask"], a["words"],
                                      a["depth"], a["status"], None)


def walk(**kw):
    a = _with(dict(target=FAKE, bf16=0, tokens=FAKE, parents=FAKE, q_start=FAKE, u=FAKE, T=8, B=2, steps=3, V=10,
                   kept=FAKE, out=FAKE, path=FAKE), kw)
    return _lib.load().dwa_verify_tree(a["target"], a["bf16"], a["tokens"], a["parents"], a["q_start"], a["u"],
                                       a["T"], a["B"], a["steps"], a["V"], a["kept"], a["out"], a["path"], None)


@pytest.mark.parametrize("kw,status", BAD_CACHE)
@pytest.mark.parametrize("call", [append, attention, keep])
def test_bad_caches(call, kw, status):
    assert call(**kw) == status, _lib.last_error()
    assert _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), BAD), (dict(T=2 ** 31), BAD), (dict(heads=0), BAD), (dict(heads=70000), SHAPE), (dict(k=None), BAD),
    (dict(v=None), BAD), (dict(slots=None), BAD), (dict(q_out=None), BAD), (dict(cos=None), BAD),
    (dict(n_positions=-1), BAD), (dict(q=FAKE + 8), SHAPE), (dict(k=FAKE + 8), SHAPE), (dict(qt=260), SHAPE),
    (dict(vh=4), SHAPE), (dict(bf16=0, kh=2), SHAPE), (dict(kt=-128), BAD), (dict(qh=-64), BAD),
    (dict(cos=FAKE + 8), SHAPE), (dict(ld_table=34), SHAPE), (dict(ld_table=28), BAD),
    (dict(tables_bf16=1, ld_table=36), SHAPE), (dict(positions=FAKE + 4), BAD), (dict(q_out=FAKE + 8), BAD),
    (dict(status=FAKE + 1), BAD),
])
def test_bad_appends(kw, status):
    assert append(**kw) == status, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(words=0), BAD), (dict(words=2 ** 21), BAD), (dict(mask=None), BAD), (dict(mask=FAKE + 4), BAD),
    (dict(max_q=65), BAD), (dict(T=-1), BAD), (dict(heads=3), SHAPE), (dict(q=None), BAD), (dict(max_q=0), BAD),
    (dict(q_start=None, T=9), BAD), (dict(q_start=None, max_q=3), BAD), (dict(scale=float("nan")), BAD),
    (dict(out=FAKE + 4), SHAPE), (dict(ld_table=2), BAD), (dict(status=FAKE + 1), BAD),
])
def test_bad_tree_attention(kw, status):
    assert attention(**kw) == status, _lib.last_error()
    assert "dwa_paged_tree_attention" in _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(layers=0), BAD), (dict(layers=70000), SHAPE), (dict(ld_layer=-8), BAD), (dict(ld_layer=4), BAD),
    (dict(B=-1), BAD), (dict(steps=0), BAD), (dict(steps=2 ** 21), SHAPE), (dict(max_pages=2 ** 28), SHAPE),
    (dict(table=None), BAD), (dict(start=None), BAD), (dict(path=None), BAD), (dict(kept=None), BAD),
    (dict(ld_table=2), BAD), (dict(path=FAKE + 2), BAD), (dict(status=FAKE + 1), BAD),
])
def test_bad_keeps(kw, status):
    assert keep(**kw) == status, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), BAD), (dict(B=-1), BAD), (dict(max_q=-1), BAD), (dict(words=0), BAD), (dict(max_q=65), BAD),
    (dict(max_q=5000, words=100), SHAPE), (dict(T=2 ** 31), SHAPE), (dict(q_start=None, T=9), BAD),
    (dict(q_start=None, max_q=3), BAD), (dict(q_start=None, B=0), BAD), (dict(parents=None), BAD),
    (dict(mask=None), BAD), (dict(depth=None), BAD), (dict(mask=FAKE + 4), BAD), (dict(status=FAKE + 2), BAD),
])
def test_bad_masks(kw, status):
    assert masks(**kw) == status, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), BAD), (dict(B=-1), BAD), (dict(steps=0), BAD), (dict(V=0), BAD), (dict(V=2 ** 30 + 1), SHAPE),
    (dict(B=2 ** 30), SHAPE), (dict(T=2 ** 31), SHAPE), (dict(q_start=None, T=9), BAD), (dict(target=None), BAD),
    (dict(tokens=None), BAD), (dict(parents=None), BAD), (dict(u=None), BAD), (dict(path=None), BAD),
    (dict(target=FAKE + 2), BAD), (dict(path=FAKE + 1), BAD),
])
def test_bad_walks(kw, status):
    assert walk(**kw) == status, _lib.last_error()


def test_empty_calls_are_noops():
    assert append(T=0, k=None) == 0 and attention(T=0, q=None) == 0 and attention(B=0, lengths=None) == 0
    assert keep(B=0, path=None) == 0 and masks(T=0, parents=None) == 0 and walk(B=0, target=None) == 0


def test_python_calls_refuse_host_tensors():
    c = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    t = torch.zeros((8, 32))
    for call in (lambda: kv_cache_append(x, x, x, t, t, c, c, i.long()),
                 lambda: paged_tree_attention(x, c, c, i[None], i, i.long()[:, None]),
                 lambda: kv_cache_keep(c, c, i[None], i[:1], i[None], i[:1]),
                 lambda: tree_masks(i),
                 lambda: verify_tree(torch.zeros(3, 8), i, i, torch.zeros(1, 2))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


class _Model:
    """What ``DWALM.verify_tree`` needs of a model; its chunk forward notes that it was called."""

    def __init__(self):
        from types import SimpleNamespace

        self.cfg, self.calls = SimpleNamespace(vocab=11), []

    def extend(self, token_ids, cache, block_table, lengths, *a, **kw):
        self.calls.append((token_ids.tolist(), lengths.tolist(), kw["parents"].tolist()))
        return torch.zeros((token_ids.shape[0], self.cfg.vocab))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _verify(model, paged, last, drafts, parents, u, **kw):
    from computd_b200.dwa_lm import DWALM

    return DWALM.verify_tree(model, last, drafts, parents, u, paged, torch.zeros((2, 4), dtype=torch.int32),
                             _i32([9, 9]), **kw)


def test_verify_tree_refuses_before_anything_is_written():
    from computd_b200 import PagedKVCache

    good = dict(last=_i32([1, 2]), drafts=_i32([[3, 4], [5, 6]]), parents=_i32([0, 1]), u=torch.zeros(2, 3))
    bad = [dict(last=_i32([1, 2, 3])), dict(last=torch.zeros(2)), dict(drafts=good["drafts"].long()),
           dict(drafts=_i32([3, 4])), dict(parents=_i32([0])), dict(parents=torch.tensor([0, 1])),
           dict(parents=_i32([[0, 1]] * 3)), dict(u=torch.zeros(2)), dict(u=torch.zeros(3, 3)),
           dict(u=torch.zeros(2, 0)), dict(u=torch.zeros(2, 3).double()), dict(u=torch.zeros(3, 2).t()),
           dict(drafts=torch.zeros((2, 4096), dtype=torch.int32), parents=torch.zeros(4096, dtype=torch.int32)),
           dict(temperature=0.0), dict(temperature=-1), dict(temperature=float("nan")), dict(temperature=1e31)]
    for kw in bad:
        model, a = _Model(), {**good, **kw}
        with pytest.raises(ValueError):
            _verify(model, PagedKVCache(1, 4, 16, 2, 16, device="cpu"), a.pop("last"), a.pop("drafts"),
                    a.pop("parents"), a.pop("u"), **a)
        assert not model.calls, kw


def test_verify_tree_step_on_the_host(monkeypatch):
    """What the chunk forward, the walk and the move are given, and what becomes of last tokens outside
    the vocabulary."""
    import computd_b200.dwa_lm as lm
    from computd_b200 import DWAError, PagedKVCache

    seen = {}

    def decide(probs, tokens, parents, u):
        seen.update(tokens=tokens.tolist(), parents=parents.tolist())
        return _i32([2, 1]), _i32([[3, 4, 7], [5, 8, -1]]), _i32([[0, 1, 2], [0, 2, -1]])

    monkeypatch.setattr(lm, "verify_tree", decide)
    for last, lost in (([1, 2], False), ([1, 11], True), ([1, -1], True)):
        model, paged = _Model(), PagedKVCache(1, 4, 16, 2, 16, device="cpu")
        monkeypatch.setattr(paged, "keep", lambda table, start, path, kept: seen.update(
            start=start.tolist(), path=path.tolist(), kept=kept.tolist()))
        got = _verify(model, paged, _i32(last), _i32([[3, 4], [12, 5]]), _i32([[0, 1], [0, 0]]), torch.zeros(2, 3))
        ids, lengths, parents = model.calls[0]
        assert ids[:4] == [1, 3, 4, min(max(last[1], 0), 10)] and ids[4:] == [10, 5] and lengths == [12, 12]
        assert parents == seen["parents"] == [-1, 0, 1, -1, 0, 0]
        assert seen["tokens"] == [1, 3, 4, last[1], 12, 5]
        assert seen["start"] == [9, 9] and seen["kept"] == [2, -1 if lost else 1]
        assert got[0].tolist() == [2, 0 if lost else 1] and got[2].tolist() == [12, 9 if lost else 11]
        assert got[1].tolist() == [[3, 4, 7], [-1] * 3 if lost else [5, 8, -1]]
        if lost:
            with pytest.raises(DWAError):
                paged.check()
        paged.check()
