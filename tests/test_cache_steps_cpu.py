"""Steps of a cache that nobody reserved, without a GPU: which pages the table names."""

from __future__ import annotations

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import experiment_config


def _cache(**kw) -> da.RoutedCache:
    return da.RoutedCache(experiment_config("qk4-s4"), 2, 3, 100, device="cpu", page_size=16, **kw)


def _named(cache: da.RoutedCache) -> list[list[int]]:
    """Pages that each sequence's row of the table names."""
    return [[page for page in row if page >= 0] for row in cache.table.tolist()]


def test_a_shared_table_names_nothing_but_a_sequences_own_pages() -> None:
    cache = _cache(pages=9)
    assert _named(cache) == [[], [], []]
    cache.advance([33, 1, 0], cache.step([33, 1, 0]))
    first, second, third = _named(cache)
    assert (len(first), len(second), len(third)) == (3, 1, 0) and len({*first, *second}) == 4
    assert cache.table[0, 3:].eq(-1).all()
    cache.release(0)
    assert _named(cache) == [[], second, []]
    cache.advance([0, 0, 80], cache.step([0, 0, 80]))
    assert _named(cache)[0] == [] and len({*_named(cache)[2], *second}) == 6
    cache.release()
    assert cache.table.eq(-1).all()


def test_sequences_with_pages_of_their_own_keep_them() -> None:
    cache = _cache()
    before = cache.table.clone()
    assert sorted(before.flatten().tolist()) == list(range(21))
    cache.release(1)
    cache.release()
    assert torch.equal(cache.table, before)


def test_no_captured_step_of_a_pool_and_none_of_uneven_counts(monkeypatch: pytest.MonkeyPatch) -> None:
    pool, own = _cache(pages=9), _cache()
    pool.advance([20, 1, 0], pool.step([20, 1, 0]))
    monkeypatch.setattr(da.RoutedCache, "_capturing", lambda cache: True)
    before = pool.table.clone()
    for counts in ([1, 1, 1], [0, 0, 0]):
        with pytest.raises(RuntimeError, match="share a pool"):
            pool.step(counts)
    with pytest.raises(RuntimeError, match="pool"):
        pool.release(0)
    assert torch.equal(pool.table, before) and pool.lengths.tolist() == [20, 1, 0]
    with pytest.raises(RuntimeError, match="as many"):
        own.step([1, 0, 1])
    assert own.step([2, 2, 2]).starts.tolist() == [0, 2, 4, 6]


def test_steps_after_replays_are_checked_against_the_devices_lengths(monkeypatch: pytest.MonkeyPatch) -> None:
    cache = _cache()
    ids = torch.zeros(3, 1, dtype=torch.long)
    cache.advance([4, 4, 4], cache.step([4, 4, 4]))
    with monkeypatch.context() as m:  # a captured step, which changes nothing here but the lengths' tensor
        m.setattr(da.RoutedCache, "_capturing", lambda cache: True)
        cache.rows(ids, None, 100)
        batch = cache.step([1, 1, 1])
        kept = cache.lengths.clone()
        cache.advance([1, 1, 1], batch)
        cache.lengths.copy_(kept)     # (nothing runs in a capture)
    cache.rows(ids.expand(3, 96), None, 100)
    cache.step([96, 96, 96])          # the four tokens that there are, and no fifth
    for _ in range(95):               # replays
        cache.lengths.add_(1)
    cache.rows(ids, None, 100)
    cache.step([1, 1, 1])
    with pytest.raises(ValueError, match="has 99 tokens"):
        cache.step([0, 2, 0])
    with pytest.raises(ValueError, match="length 101"):
        cache.rows(ids.expand(3, 2), None, 100)
    cache.advance([1, 0, 0], cache.step([1, 0, 0]))
    assert cache.lengths.tolist() == [100, 99, 99]
    with pytest.raises(ValueError, match="has 100 tokens"):
        cache.step([1, 1, 1])
    cache.release(0)
    assert cache.step([100, 1, 1]).max_new == 100


@pytest.mark.parametrize("pages", [None, 9])
def test_a_step_made_before_a_capture_that_counts_it_in(pages, monkeypatch: pytest.MonkeyPatch) -> None:
    cache = _cache(pages=pages)
    batch = cache.step([2, 2, 2])
    with monkeypatch.context() as m:
        m.setattr(da.RoutedCache, "_capturing", lambda cache: True)
        cache.advance([2, 2, 2], batch)  # (counts on the CPU at once, as a replay does)
    assert cache.lengths.tolist() == [2, 2, 2]
    with pytest.raises(ValueError, match="has 2 tokens"):
        cache.step([99, 0, 0])
