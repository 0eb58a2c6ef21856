"""Host logic of the paged cache and of the scores, without a GPU: pages handed out and given back, steps, refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import _lib, experiment_config


def _cache(**kw) -> da.RoutedCache:
    return da.RoutedCache(experiment_config("qk4-s4"), 2, 3, 100, device="cpu", **kw)


def test_every_sequence_owns_its_pages() -> None:
    cache = _cache(page_size=16)
    assert cache.key_pages.shape == (2, 21, 16, 4, 128) and cache.value_pages.shape == (2, 21, 16, 512)
    assert sorted(cache.table.flatten().tolist()) == list(range(21))
    batch = cache.step([5, 5, 5])
    assert batch.starts.tolist() == [0, 5, 10, 15] and batch.max_new == 5 and batch.starts.dtype == torch.int32
    assert cache.positions(batch, [5, 5, 5], 100).tolist() == [0, 1, 2, 3, 4] * 3
    cache.advance([5, 5, 5], batch)
    batch = cache.step([1, 0, 4])
    assert batch.starts.tolist() == [0, 1, 1, 5]
    assert cache.positions(batch, [1, 0, 4], 8).tolist() == [5, 5, 6, 7, 7]  # (clamped)
    cache.advance([1, 0, 4], batch)
    assert cache.lengths.tolist() == [6, 5, 9]
    cache.release(1)
    assert cache.lengths.tolist() == [6, 0, 9]


def test_a_shared_pool() -> None:
    cache = _cache(page_size=16, pages=5)
    batch = cache.step([33, 1, 0])
    owned = cache.table[0, :3].tolist() + cache.table[1, :1].tolist()
    assert len(set(owned)) == 4
    cache.advance([33, 1, 0], batch)
    with pytest.raises(RuntimeError, match="1 left"):
        cache.step([0, 16, 1])
    cache.step([0, 15, 0])  # fits the page that it has
    cache.release(0)
    batch = cache.step([0, 15, 64])
    assert not set(cache.table[2, :4].tolist()) & {cache.table[1, 0].item()} and len(set(cache.table[2, :4].tolist())) == 4
    assert cache.lengths.tolist() == [0, 1, 0]


def test_cache_refusals() -> None:
    config = experiment_config("a1")
    for bad in ({"page_size": 24}, {"page_size": 8}, {"dtype": torch.float32}, {"pages": 0}):
        with pytest.raises(ValueError):
            da.RoutedCache(config, 1, 1, 10, device="cpu", **bad)
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            da.RoutedCache(config, *sizes, device="cpu")
    with pytest.raises(ValueError, match="causal"):
        da.RoutedCache(experiment_config("a1", causal=False), 1, 1, 1, device="cpu")
    cache = _cache()
    for counts in ([1, 1], [1, 1, -1]):
        with pytest.raises(ValueError):
            cache.step(counts)
    with pytest.raises(ValueError, match="exceed"):
        cache.step([101, 0, 0])
    ids = torch.zeros(3, 4, dtype=torch.long)
    assert cache.rows(ids, None, 100)[1] == [4, 4, 4]
    assert cache.rows(ids[0], [4, 0, 0], 100)[0].shape == (4,)
    for bad, counts in ((ids[:2], None), (ids[0], None), (ids[0], [1, 1, 1])):
        with pytest.raises(ValueError):
            cache.rows(bad, counts, 100)
    with pytest.raises(ValueError, match="maximum"):
        cache.rows(ids, None, 3)


def test_calls_on_cpu_tensors_are_refused() -> None:
    cache = _cache(page_size=16)
    batch = cache.step([1, 1, 1])
    k, v = torch.zeros(4, 3, 128, dtype=torch.bfloat16), torch.zeros(3, 512, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        da.append_paged(k, v, *cache.layer(0), batch)
    with pytest.raises(ValueError, match="CUDA"):
        da.routed_attention_paged(k, *cache.layer(0), batch, torch.ones(4), torch.ones(4))
    with pytest.raises(ValueError, match="at least one page"):
        da.append_paged(k, v, *cache.layer(0), batch._replace(table=batch.table[:, :0]))
    with pytest.raises(ValueError, match="CUDA"):
        da.token_log_probs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))


def test_entry_points_check_on_the_host() -> None:
    handle = _lib.lib()
    one = ctypes.create_string_buffer(64)
    p = ctypes.addressof(one) & ~15

    def append(page=16, dtype=_lib.DA_BF16, r=64, keys=p, tokens=0, pages=4):
        return handle.da_paged_append(keys, _lib.DA_BF16, 64, 64, p, _lib.DA_BF16, 128, tokens, p, p, dtype, pages, page, 1, r, 128, p,
                                      1, 1, p, p, 1, p, None)

    assert append() == _lib.DA_OK  # no tokens: nothing to do
    assert append(keys=None) == _lib.DA_ERR_NULL
    assert append(page=24) == append(r=12) == append(pages=0) == append(pages=2**31) == _lib.DA_ERR_SHAPE
    assert append(dtype=_lib.DA_F32) == _lib.DA_ERR_DTYPE

    def attend(page=16, dtype=_lib.DA_BF16, r=64, d=128, maps=1, q=p, stride=64, weights=p, tokens=0):
        return handle.da_paged_attn(q, 64, stride, tokens, p, p, dtype, 4, page, 1, r, d, maps, p, 1, 1, p, p, 1, 0, p, weights, 0, 0, p,
                                    None, 0, p, None)

    assert attend() == _lib.DA_OK
    assert attend(q=None) == attend(maps=2, weights=None) == _lib.DA_ERR_NULL
    assert attend(page=8) == _lib.DA_ERR_SHAPE
    assert attend(r=96) == attend(d=64) == attend(maps=5) == attend(r=512, maps=2) == _lib.DA_ERR_UNSUPPORTED
    assert attend(stride=66) == attend(q=p + 2) == _lib.DA_ERR_ALIGN
    assert attend(dtype=_lib.DA_F32) == _lib.DA_ERR_DTYPE
    assert handle.da_paged_attn_workspace_size(0, 1, 4, 16, 1, 1, 64, 128, 1, 0) == 0
    assert handle.da_paged_attn_workspace_size(1, 1, 4, 16, 1, 1, 96, 128, 1, 0) == -1
    assert handle.da_paged_attn_workspace_size(4096, 4, 64, 64, 2048, 4, 128, 512, 4, 0) > 0
    assert handle.da_token_log_probs(p, _lib.DA_F32, 4, 1, 4, p, 5, p, p, p, p, None, None) == _lib.DA_ERR_SHAPE
    assert handle.da_token_log_probs(p, _lib.DA_F32, 4, 1, 4, p, 1, p, p, None, None, None, None) == _lib.DA_ERR_NULL
    assert handle.da_token_log_probs(p, 7, 4, 1, 4, p, 0, p, p, None, None, None, None) == _lib.DA_ERR_DTYPE
    assert handle.da_token_log_probs(None, _lib.DA_F32, 4, 0, 4, None, 0, None, None, None, None, None, None) == _lib.DA_OK
    assert handle.da_token_log_probs_bwd(p, _lib.DA_F32, 4, 1, 4, p, None, p, p, p, p, 4, None) == _lib.DA_ERR_NULL
