"""What the language model's cache and scores refuse before anything runs, without a GPU."""

from __future__ import annotations

import pytest

from double_attention_b200 import DoubleAttentionLM, experiment_config


def test_a_cache_of_no_positions_is_refused() -> None:
    lm = DoubleAttentionLM(64, 40, experiment_config("a1"), 1)
    with pytest.raises(ValueError, match="at least one"):
        lm.new_cache(2, 0)
    assert lm.new_cache(2).max_length == 40 and lm.new_cache(2, 7).max_length == 7
