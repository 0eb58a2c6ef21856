"""Scores of few tokens by the models: fewer positions than the attention's smallest tile has.

Tolerances, fixed before the first run: the same sequences in a wider batch go through other splits of the same sums, with
roundings to bf16 that differ: logits agree to 0.1 of their spread, sqrt(512), and half a step of bf16 on each side (2^-7 of
the value), as through the cache; a log probability is a logit less a mean of others, twice that.  Gradients agree to a cosine
of 0.999.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import double_attention_b200 as da
from double_attention_b200 import DoubleAttentionLM, experiment_config, ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
SPREAD = 512**0.5
SIZES = [(1, 2), (1, 40), (4, 2), (3, 22), (2, 64), (1, 128), (127, 2), (1, 129)]


def _lm(preset: str, positions: int = 400, **overrides) -> DoubleAttentionLM:
    torch.manual_seed(0)
    return DoubleAttentionLM(512, positions, experiment_config(preset, **overrides), 2, feedforward_dim=1536).cuda().eval()


def _ids(batch: int, length: int, seed: int = 1) -> torch.Tensor:
    return torch.randint(0, 512, (batch, length), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    assert got.shape == want.shape and got.isfinite().all()
    assert ((got.double() - want.double()).abs() <= 0.2 * SPREAD + 2.0**-6 * want.double().abs()).all()


@pytest.mark.parametrize(("preset", "overrides"), [("a1", {}), ("qk4-s4", {}), ("qk2-s2", {"map_combine": "concat"})])
@pytest.mark.parametrize(("batch", "length"), SIZES)
def test_short_sequences_are_scored(preset, overrides, batch, length) -> None:
    lm, ids = _lm(preset, **overrides), _ids(batch, length)
    others = torch.cat((ids, _ids(160, length, 2)))
    with torch.autocast("cuda", dtype=BF16):
        made, wide = lm.score(ids, top=3), lm.score(others, top=3)
        assert made.log_probs.shape == made.entropy.shape == (batch, length - 1) and made.top_tokens.shape == (batch, length - 1, 3)
        _near(made.log_probs, wide.log_probs[:batch])
        _near(made.top_log_probs, wide.top_log_probs[:batch])
        loss, other = -made.log_probs.sum() - made.entropy.sum(), -wide.log_probs[:batch].sum() - wide.entropy[:batch].sum()
    loss.backward()
    mine = {name: p.grad.clone() for name, p in lm.named_parameters() if p.grad is not None}
    lm.zero_grad()
    other.backward()
    assert mine.keys() == {name for name, p in lm.named_parameters() if p.grad is not None}
    for name, p in lm.named_parameters():
        if name in mine and p.grad.abs().max() > 1e-6 * SPREAD:  # (a single position's query and key have none)
            assert F.cosine_similarity(mine[name].flatten().double(), p.grad.flatten().double(), dim=0) >= 0.999, name
    assert ops.device_status() == 0


@pytest.mark.parametrize(("batch", "length"), SIZES)
def test_short_sequences_are_scored_in_int8(batch, length) -> None:
    served, ids = da.Int8DoubleAttentionLM(_lm("a1")), _ids(batch, length)
    made, wide = served.score(ids, top=3), served.score(torch.cat((ids, _ids(160, length, 2))), top=3)
    _near(made.log_probs, wide.log_probs[:batch])
    assert made.top_tokens.shape == (batch, length - 1, 3)


def test_a_model_of_few_positions_is_scored() -> None:
    lm = _lm("a1", positions=20)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        made = lm.score(_ids(1, 21))
        assert made.log_probs.shape == (1, 20) and made.log_probs.isfinite().all()
        with pytest.raises(ValueError, match="maximum"):
            lm.score(_ids(1, 22))
        assert lm.score(_ids(1, 5)[:0]).log_probs.shape == (0, 4)


def test_an_int8_model_that_sees_later_tokens_is_not_scored() -> None:
    with pytest.raises(ValueError, match="causal"):
        da.Int8DoubleAttentionLM(_lm("a1", causal=False)).score(_ids(2, 10))
