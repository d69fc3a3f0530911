"""CPU: the host side of the serving calls: where new tokens go."""
import pytest
import torch

from computd_b200 import PagedKVCache


def _cache(n_pages=40, page_size=16):
    return PagedKVCache(1, n_pages, page_size, 2, 16, device="cpu")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _slots_by_rows(cache, table, lengths, q_start, n):
    """The definition, row by row."""
    out = []
    for row in range(n):
        slot = -1
        for b in range(len(lengths)):
            if q_start[b] <= row < q_start[b + 1]:
                position = lengths[b] - (q_start[b + 1] - row)
                if 0 <= position < len(table[b]) * cache.page_size:
                    page = table[b][position // cache.page_size]
                    slot = page * cache.page_size + position % cache.page_size if page >= 0 else -2
        out.append(slot)
    return out


@pytest.mark.parametrize("q_start", [[0, 3, 3, 10, 12], [2, 3, 7, 7, 9], [5, 5, 5, 5, 5], [4, 9, 9, 30, 30],
                                     [3, 3, 4, 8, 20]])
def test_slots_of_rows_in_and_outside_every_sequence(q_start):
    """Rows before the first sequence's and behind the last one's have no slot; neither have new
    tokens that the length leaves no place for."""
    cache = _cache()
    table = torch.randperm(40, generator=torch.Generator().manual_seed(0))[:16].view(4, 4).tolist()
    lengths = [40, 0, 17, 64]
    slots, positions = cache.slots(_i32(table), _i32(lengths), _i32(q_start), 24)
    assert slots.dtype == torch.int64 and positions.dtype == torch.int64
    assert slots.tolist() == _slots_by_rows(cache, table, lengths, q_start, 24)
    assert int(positions.min()) >= 0 and int(positions.max()) < 64


def test_slots_on_bad_pages_are_not_skipped():
    """A negative page number gives a slot that the write reports (-1 would pass it over in silence);
    one behind the last page gives one outside the cache."""
    cache = _cache()
    table = [[-1, 7, -3, 40]]
    slots, _ = cache.slots(_i32(table), _i32([64]), _i32([0, 64]), 64)
    assert slots.tolist() == _slots_by_rows(cache, table, [64], [0, 64], 64)
    assert bool((slots[:16] == -2).all()) and bool((slots[32:48] == -2).all())
    assert bool((slots[16:32] == 7 * 16 + torch.arange(16)).all()) and int(slots[48:].min()) >= 40 * 16


def test_row_counts_are_planned_for_a_few():
    from computd_b200.dwa_lm import plan_rows

    counts = [plan_rows(t) for t in range(1, 65537)]
    assert all(c >= t for t, c in enumerate(counts, 1)) and counts == sorted(counts)
    assert len(set(counts)) == 63
    assert all(plan_rows(c) == c for c in set(counts))
    assert [plan_rows(t) for t in (0, 1, 2, 3, 64, 65, 128, 129, 1024, 1025)] == \
        [1, 1, 2, 4, 64, 128, 128, 256, 1024, 1152]
    assert all(8 * (c - t) <= t for t, c in enumerate(counts, 1) if t > 1024)


class _Model:
    """What ``DWALM.verify`` needs of a model; its chunk forward notes that it was called."""

    def __init__(self, vocab=11):
        from types import SimpleNamespace

        self.cfg, self.calls = SimpleNamespace(vocab=vocab), []

    def extend(self, token_ids, cache, block_table, lengths, *a, **kw):
        self.calls.append((token_ids.tolist(), lengths.tolist()))
        return torch.zeros((token_ids.shape[0], self.cfg.vocab))


def _verify(model, cache, last, drafts, **kw):
    from computd_b200.dwa_lm import DWALM

    B, K = drafts.shape
    a = dict(draft_probs=None, accept_u=torch.zeros(B, K), sample_u=torch.zeros(B), temperature=1.0,
             draft_lengths=None)
    a.update(kw)
    return DWALM.verify(model, last, drafts, a.pop("draft_probs"), a.pop("accept_u"), a.pop("sample_u"), cache,
                        torch.zeros((B, 4), dtype=torch.int32), torch.full((B,), 9, dtype=torch.int32), **a)


@pytest.mark.parametrize("temperature", [0, 0.0, -1.0, float("nan"), float("inf"), 1e-46])
def test_verify_refuses_temperatures(temperature):
    model = _Model()
    with pytest.raises(ValueError, match="temperature"):
        _verify(model, _cache(), _i32([1, 2]), _i32([[3, 4], [5, 6]]), temperature=temperature)
    assert not model.calls


def test_verify_refuses_before_anything_is_written():
    """What verify_drafts would refuse afterwards, with the chunk already in the cache."""
    good = dict(last=_i32([1, 2]), drafts=_i32([[3, 4], [5, 6]]))
    bad = [dict(drafts=good["drafts"].long()), dict(drafts=good["drafts"].float()), dict(drafts=_i32([3, 4])),
           dict(last=_i32([1, 2, 3])), dict(last=torch.zeros(2)), dict(accept_u=torch.zeros(2, 3)),
           dict(accept_u=torch.zeros(2, 2).double()), dict(sample_u=torch.zeros(3)),
           dict(draft_probs=torch.zeros(2, 2, 12)), dict(draft_probs=torch.zeros(2, 2, 11).bfloat16()),
           dict(draft_probs=torch.zeros(2, 11, 2).transpose(1, 2)), dict(draft_lengths=torch.zeros(2)),
           dict(draft_lengths=_i32([1]))]
    for kw in bad:
        model, a = _Model(), {**good, **kw}
        with pytest.raises(ValueError):
            _verify(model, _cache(), a.pop("last"), a.pop("drafts"), **a)
        assert not model.calls, kw


def test_verify_reports_last_tokens_outside_the_vocabulary(monkeypatch):
    """Their sequences get no tokens and stay as long as they were, and the cache's status says so;
    the others go on."""
    import computd_b200.dwa_lm as lm
    from computd_b200 import DWAError

    def decide(probs, drafts, *a, **kw):
        B, K = drafts.shape
        return torch.arange(B, dtype=torch.int32) % (K + 1), torch.full((B, K + 1), 5, dtype=torch.int32)

    monkeypatch.setattr(lm, "verify_drafts", decide)
    for last, bad in (([1, -1, 10, 11, 2 ** 31 - 1], [1, 3, 4]), ([0, 10, 3, 4, 5], [])):
        model, cache = _Model(), _cache()
        accepted, tokens, lengths = _verify(model, cache, _i32(last), torch.full((5, 3), 2, dtype=torch.int32))
        ids, asked = model.calls[0]
        assert asked == [13] * 5 and all(0 <= x < 11 for x in ids)
        for b in range(5):
            assert accepted[b] == (0 if b in bad else b % 4)
            assert tokens[b].tolist() == ([-1] * 4 if b in bad else [5] * 4)
            assert lengths[b] == (9 if b in bad else 10 + b % 4)
        assert lengths.dtype == accepted.dtype == tokens.dtype == torch.int32
        if bad:
            with pytest.raises(DWAError):
                cache.check()
        cache.check()


@pytest.mark.parametrize("made,used", [(True, False), (False, True), (True, True)])
def test_a_cache_serves_in_and_out_of_inference_mode(made, used):
    from computd_b200 import DWAError

    with torch.inference_mode(made):
        cache = _cache()
    with torch.inference_mode(used):
        cache.report(torch.tensor([False, True]))
        with pytest.raises(DWAError):
            cache.check()
        cache.check()
