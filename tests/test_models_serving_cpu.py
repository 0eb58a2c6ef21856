"""What the language model's cache and scores refuse before anything runs, without a GPU."""

from __future__ import annotations

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import DoubleAttentionLM, experiment_config


def test_a_cache_of_no_positions_is_refused() -> None:
    lm = DoubleAttentionLM(64, 40, experiment_config("a1"), 1)
    with pytest.raises(ValueError, match="at least one"):
        lm.new_cache(2, 0)
    assert lm.new_cache(2).max_length == 40 and lm.new_cache(2, 7).max_length == 7


def test_scores_of_an_attention_that_sees_later_tokens_are_refused() -> None:
    lm = DoubleAttentionLM(64, 40, experiment_config("a1", causal=False), 1)
    with pytest.raises(ValueError, match="causal"):
        lm.score(torch.zeros(2, 10, dtype=torch.long))


def test_an_output_over_the_inputs_is_refused() -> None:
    """(On CPU tensors, which the next check refuses: nothing is launched.)"""
    pages = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16), torch.zeros(3, 16, 128, dtype=torch.bfloat16)[:2]
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    batch = da.PagedBatch(table, one, torch.tensor([0, 8], dtype=torch.int32), 8)
    room = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    query = room[1:2]
    for out in (room[1], query[0], pages[0][1, 8:, 0], pages[1][0, :8], room.flatten()[1000 * 2:1000 * 2 + 1024].view(8, 128)):
        assert out.data_ptr() % 16 == 0
        with pytest.raises(ValueError, match="shares memory"):
            da.routed_attention_paged(query, *pages, batch, torch.ones(1), out=out)
    for out in (room[0], room[2], torch.empty(8, 128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="CUDA"):
            da.routed_attention_paged(query, *pages, batch, torch.ones(1), out=out)
