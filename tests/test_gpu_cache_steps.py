"""Steps of a cache on the GPU that nobody reserved: reported, and nothing of another sequence is written."""

from __future__ import annotations

import pytest
import torch

from double_attention_b200 import DoubleAttentionLM, Int8DoubleAttentionLM, append_paged, experiment_config, ops, paged, routed_attention_paged

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _lm(preset: str = "a1", positions: int = 400) -> DoubleAttentionLM:
    torch.manual_seed(0)
    return DoubleAttentionLM(512, positions, experiment_config(preset), 2, feedforward_dim=1536).cuda().eval()


def _ids(batch: int, length: int, seed: int = 1) -> torch.Tensor:
    return torch.randint(0, 512, (batch, length), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


@pytest.mark.parametrize("new", [1, 40])
def test_a_step_past_a_sequences_pages_writes_nothing(new) -> None:
    """A batch used for a second step, whose tokens no page was reserved for."""
    config = experiment_config("a1")
    cache = paged.RoutedCache(config, 1, 2, 400, page_size=16, pages=12)
    cache.advance([32, 32], cache.step([32, 32]))  # two pages each, full
    keys = torch.randn(1, 2 * new, config.routing_dim, device="cuda").to(BF16)
    values = torch.randn(2 * new, 512, device="cuda").to(BF16)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    cache.table[1, 2:5] = torch.tensor([9, 10, 11], dtype=torch.int32)  # (the second sequence has pages for them)
    batch = paged.PagedBatch(cache.table, cache.lengths, starts, new)
    before = [t.clone() for t in cache.layer(0)]
    append_paged(keys, values, *cache.layer(0), batch)
    assert ops.device_status() == paged.BAD_PAGE
    written = torch.zeros(12, dtype=torch.bool, device="cuda")
    written[9:9 + -(-new // 16)] = True
    for now, was in zip(cache.layer(0), before):
        assert torch.equal(now[~written], was[~written]) and not torch.equal(now[written], was[written])
    y = routed_attention_paged(keys, *cache.layer(0), batch, torch.tensor([16.0], device="cuda"))
    assert ops.device_status() == paged.BAD_PAGE
    assert y[:new].isnan().all() and y[new:].isfinite().all()


def test_a_released_sequences_pages_are_another_ones() -> None:
    lm, ids = _lm(), _ids(2, 100)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        cache = lm.new_cache(2, page_size=16, pages=7)
        lm.extend(ids[0], cache, [100, 0])
        cache.release(0)
        want = lm.extend(ids[1], cache, [0, 100])
        assert ops.device_status() == 0
        # the first sequence's old entries lead nowhere
        stale = paged.PagedBatch(cache.table, torch.tensor([50, 0], dtype=torch.int32, device="cuda"),
                                 torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda"), 1)
        before = [t.clone() for t in cache.layer(0)]
        key = torch.randn(1, 1, lm.stack.config.routing_dim, device="cuda").to(BF16)
        append_paged(key, torch.randn(1, 512, device="cuda").to(BF16), *cache.layer(0), stale)
        assert ops.device_status() == paged.BAD_PAGE
        assert all(torch.equal(now, was) for now, was in zip(cache.layer(0), before))
        cache.release()
        again = lm.extend(ids[1], cache, [0, 100])
    assert torch.equal(want, again)


def test_steps_that_replays_cannot_follow_are_not_captured() -> None:
    lm, ids = _lm(), _ids(2, 3)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, cache_enabled=False):
        pool, own = lm.new_cache(2, page_size=16, pages=7), lm.new_cache(2)
        lm.extend(ids, pool)
        lm.extend(ids, own)
        pool.release()
        refused = []
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            for call in (lambda: lm.extend(ids, pool), lambda: pool.release(), lambda: lm.extend(ids[0], own, [1, 2])):
                try:
                    call()
                except RuntimeError as error:
                    refused.append(str(error))
        assert len(refused) == 3 and "pool" in refused[0] and "pool" in refused[1] and "as many" in refused[2]
        # (the capture went on, and the caches are as they were)
        assert own.lengths.tolist() == [3, 3] and pool.lengths.tolist() == [0, 0]
        want = lm.new_cache(2)
        assert torch.equal(lm.extend(ids, pool), lm.extend(ids, want))
    assert ops.device_status() == 0


def test_eager_steps_after_replays_know_the_length() -> None:
    lm, ids = _lm(positions=64), _ids(2, 64)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, cache_enabled=False):
        cache, other = lm.new_cache(2), lm.new_cache(2)
        token = ids[:, :1].clone()
        lm.extend(token, cache)
        cache.release()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lm.extend(token, cache)
        for i in range(60):
            token.copy_(ids[:, i:i + 1])
            graph.replay()
        with pytest.raises(ValueError, match="length 65 exceeds"):
            lm.extend(ids[:, 59:], cache)
        last = lm.extend(ids[:, 60:], cache)
        want = lm.extend(ids, other)[:, 60:]
        assert cache.lengths.tolist() == [64, 64]
        with pytest.raises(ValueError, match="exceeds"):
            lm.extend(token, cache)
    # (as through the cache in one step or several: roundings to bf16 differ, 0.1 of the logits' spread and half a step each)
    assert ((last.double() - want.double()).abs() <= 0.1 * 512**0.5 + 2.0**-7 * want.double().abs()).all()
    assert ops.device_status() == 0


def _status(stream: torch.cuda.Stream) -> int:
    """What calls captured on ``stream`` have reported."""
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        return ops.device_status()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize(("positions", "most"), [(400, 40), (40, None), (40, 64), (64, 64)])
@pytest.mark.parametrize("new", [1, 3, 20])
def test_replays_past_the_last_position_are_reported(new, positions, most, int8) -> None:
    """Of two sequences the longer one runs past the most positions: NaN and a status, and the other goes on."""
    lm = _lm(positions=positions)
    lm, limit = Int8DoubleAttentionLM(lm) if int8 else lm, min(positions, most or positions)
    ids = _ids(2, new, 3)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, cache_enabled=False):
        cache, other = lm.new_cache(2, most), lm.new_cache(2, most)
        lm.extend(ids, cache)
        cache.release()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            logits = lm.extend(ids, cache)
        first = _ids(1, limit - 2 * new)[0]
        for c in (cache, other):  # two more steps fit the second sequence
            lm.extend(first, c, [0, limit - 2 * new])
        for _ in range(2):
            graph.replay()
            want = lm.extend(ids, other)
            assert ((logits.double() - want.double()).abs() <= 0.1 * 512**0.5 + 2.0**-7 * want.double().abs()).all()
            assert _status(stream) == 0
        before = [t.clone() for t in (cache.key_pages, cache.value_pages)]
        graph.replay()
        assert _status(stream) == paged.BAD_PAGE
        want = lm.extend(ids[0], other, [new, 0]) if limit >= 3 * new else None
    assert logits[1].isnan().all()
    if want is not None:
        assert ((logits[0].double() - want.double()).abs() <= 0.1 * 512**0.5 + 2.0**-7 * want.double().abs()).all()
    own = cache.table[1].long()  # nothing of the second sequence is written
    for now, was in zip((cache.key_pages, cache.value_pages), before):
        assert torch.equal(now[:, own], was[:, own])
