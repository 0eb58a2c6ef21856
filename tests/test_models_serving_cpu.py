"""What the language model's cache and scores refuse before anything runs, without a GPU."""

from __future__ import annotations

import pytest
import torch

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
