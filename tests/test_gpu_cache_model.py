"""The operators over a paged cache and the scores together, as a model uses them: prompts taken in chunks, tokens decoded
one by one, uneven batches, a shared pool of pages, a captured step, and scores of tokens with their gradient.

Tolerances, fixed from the formats: a step through the cache computes what a forward over the whole sequences does, with
other splits of the same fp32 sums and its softmax weights rounded against another offset: roundings to bf16 (2^-8 each, a
few dozen in random directions, 0.02 of a value's spread) differ, so logits agree to a cosine of 0.999 and, over 1e5 of them,
to 0.1 of their spread.  That is sqrt(512): the head is the token embedding, normal entries against normalised rows of 512.
Each side rounds its own logits to bf16, half a step (2^-8 of the value) each.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import double_attention_b200 as da
from double_attention_b200 import DoubleAttentionLM, experiment_config, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SPREAD = 512**0.5


def _lm(preset: str = "a1", layers: int = 2, **overrides) -> DoubleAttentionLM:
    torch.manual_seed(0)
    return DoubleAttentionLM(512, 400, experiment_config(preset, **overrides), layers, feedforward_dim=1536).cuda().eval()


def _ids(batch: int, length: int, seed: int = 1) -> torch.Tensor:
    return torch.randint(0, 512, (batch, length), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    assert got.shape == want.shape and got.isfinite().all()
    assert F.cosine_similarity(got.double().flatten(), want.double().flatten(), dim=0) >= 0.999
    assert ((got.double() - want.double()).abs() <= 0.1 * SPREAD + 2.0**-7 * want.double().abs()).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize(("preset", "overrides"), [("a1", {}), ("qk4-s4", {}), ("qk2-s1", {}), ("qk1-s2", {}),
                                                   ("qk2-s2", {"map_combine": "concat"}), ("a1-silu", {}), ("a1-r512-d512", {})])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_chunks_and_tokens_give_the_whole_sequences_logits(preset, overrides, dtype) -> None:
    lm, ids = _lm(preset, **overrides), _ids(2, 203)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        want = lm(ids)[0]
        cache = lm.new_cache(2, dtype=dtype, page_size=32)
        got, at = [], 0
        for n in (1, 130, 5, 64, 1, 1, 1):
            got.append(lm.extend(ids[:, at:at + n], cache))
            at += n
    assert cache.lengths.tolist() == [203, 203]
    _near(torch.cat(got, 1), want)


@pytest.mark.parametrize("preset", ["a1", "qk4-s4"])
def test_uneven_sequences_in_a_shared_pool(preset) -> None:
    lm, ids = _lm(preset), _ids(3, 300)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        want = lm(ids)[0]
        cache = lm.new_cache(3, page_size=16, pages=30)
        held = [0, 0, 0]
        for counts in ([200, 0, 7], [1, 33, 1], [1, 1, 0], [60, 2, 150]):
            packed = torch.cat([ids[b, h:h + n] for b, (h, n) in enumerate(zip(held, counts))])
            got = lm.extend(packed, cache, counts)
            _near(got, torch.cat([want[b, h:h + n] for b, (h, n) in enumerate(zip(held, counts))]))
            held = [h + n for h, n in zip(held, counts)]
        assert cache.lengths.tolist() == held
        with pytest.raises(RuntimeError, match="pages"):
            lm.extend(_ids(3, 40).flatten(), cache, [40, 40, 40])
        cache.release(0)
        _near(lm.extend(ids[0, :100], cache, [100, 0, 0]), want[0, :100])  # into pages that others had
        cache.release()
        assert cache.lengths.tolist() == [0, 0, 0]
        _near(lm.extend(ids[:, :150], cache), want[:, :150])


def test_a_captured_step() -> None:
    lm, ids = _lm("qk4-s4"), _ids(4, 20)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, cache_enabled=False):
        want = lm(_wide(ids))[0][:, :20]
        cache = lm.new_cache(4)
        token = ids[:, :1].clone()
        lm.extend(token, cache)
        cache.release()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = lm.extend(token, cache)
        cache.lengths.zero_()
        got = []
        for i in range(20):
            token.copy_(ids[:, i:i + 1])
            graph.replay()
            got.append(logits.clone())
    assert cache.lengths.tolist() == [20] * 4
    _near(torch.cat(got, 1), want)


def _wide(ids: torch.Tensor) -> torch.Tensor:
    """The ids and more behind them: a forward wants 128 rows."""
    return torch.cat((ids, _ids(ids.shape[0], 60, 9)), 1)


@pytest.mark.parametrize(("preset", "overrides"), [("a1", {}), ("qk4-s4", {}), ("qk2-s2", {"map_combine": "concat"})])
def test_int8_model_through_a_cache(preset, overrides) -> None:
    served, ids = da.Int8DoubleAttentionLM(_lm(preset, **overrides)), _ids(3, 150)
    want = served(ids)
    cache = served.new_cache(3)
    got = [served.extend(ids[:, :140], cache)] + [served.extend(ids[:, i:i + 1], cache) for i in range(140, 150)]
    _near(torch.cat(got, 1), want)
    uneven = served.new_cache(3, page_size=128)
    _near(served.extend(torch.cat((ids[0, :150], ids[2, :9])), uneven, [150, 0, 9]), torch.cat((want[0], want[2, :9])))


def test_scores_of_a_models_tokens() -> None:
    lm, ids = _lm(), _ids(3, 131)
    with torch.autocast("cuda", dtype=BF16):
        made = lm.score(ids, top=5)
        logits = lm(ids[:, :-1])[0]
        other = F.cross_entropy(logits.float().flatten(0, 1), ids[:, 1:].flatten())  # (of 16-bit logits it is 7e-5 off itself)
    lp = torch.log_softmax(logits.double(), -1)
    assert made.log_probs.shape == made.entropy.shape == (3, 130) and made.top_tokens.shape == (3, 130, 5)
    want = lp.gather(-1, ids[:, 1:, None])[..., 0]
    assert ((made.log_probs - want).abs() <= 4e-6 * (1 + want.abs())).all()
    assert torch.equal(made.top_tokens, torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :5])
    loss = -made.log_probs.mean()
    assert abs(loss.item() - other.item()) <= 1e-5 * other.item()
    loss.backward()
    mine = {name: p.grad.clone() for name, p in lm.named_parameters() if p.grad is not None}
    lm.zero_grad()
    other.backward()
    for name, p in lm.named_parameters():
        if p.grad is not None:
            assert F.cosine_similarity(mine[name].flatten().double(), p.grad.flatten().double(), dim=0) >= 0.999, name
    served = da.Int8DoubleAttentionLM(lm)
    scored = served.score(ids, top=1)
    assert torch.equal(scored.top_tokens[..., 0], served(ids[:, :-1]).float().argmax(-1))


def test_decoding_greedily_and_scoring_agree() -> None:
    """A run as a server makes it: a prompt, tokens by the likeliest alternative, then the whole scored at once."""
    lm, prompt = _lm("qk2-s2"), _ids(2, 100)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        cache = lm.new_cache(2)
        logits = lm.extend(prompt, cache)[:, -1]
        tokens, scores = [], []
        for _ in range(30):
            best = da.token_log_probs(logits, logits.argmax(-1), top=1)
            tokens.append(best.top_tokens)
            scores.append(best.log_probs)
            assert torch.equal(best.log_probs, best.top_log_probs[:, 0])
            logits = lm.extend(best.top_tokens, cache)[:, -1]
        whole = lm.score(torch.cat((prompt, *tokens), 1))
    assert (whole.log_probs[:, 99:] - torch.stack(scores, 1)).abs().max() <= 0.1 * SPREAD


def test_refusals() -> None:
    lm, ids = _lm(), _ids(2, 10)
    with torch.autocast("cuda", dtype=BF16):
        cache = lm.new_cache(2, max_length=64)
        for bad, counts in ((ids[:1], None), (ids[0], None), (ids[0], [5, 6]), (ids.flatten(), [20, -1, 1])):
            with pytest.raises(ValueError):
                lm.extend(bad, cache, counts)
        with pytest.raises(ValueError, match="exceed"):
            lm.extend(_ids(2, 65), cache)
        with pytest.raises(ValueError, match="exceeds configured maximum"):
            lm.extend(_ids(2, 401), lm.new_cache(2, max_length=500))
        with pytest.raises(ValueError, match="computes in"):
            lm.extend(ids, lm.new_cache(2, dtype=FP16))
        assert cache.lengths.tolist() == [0, 0]
        assert lm.extend(ids[:, :0], cache).shape == (2, 0, 512)
        attention = lm.stack.blocks[0].attention
        step = cache.step([1, 1])
        with pytest.raises(ValueError, match="packed"):
            attention(torch.randn(2, 1, 512, device="cuda"), bank=lm.stack.banks[0], cache=(*cache.layer(0), step))
        with pytest.raises(RuntimeError, match="no backward"):  # training through a cache
            attention(torch.randn(1, 2, 512, device="cuda"), bank=lm.stack.banks[0], cache=(*cache.layer(0), step))
        with pytest.raises(ValueError, match="T at least 2"):
            lm.score(ids[:, :1])
    with pytest.raises(ValueError, match="causal"):
        DoubleAttentionLM(64, 32, experiment_config("a1", causal=False), 1).cuda().new_cache(1)
