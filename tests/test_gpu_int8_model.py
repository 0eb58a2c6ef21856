"""The eight-bit operators together: the language model served in int8, and trained with its feed-forward
activations kept in 8 bits.

Tolerances, fixed from the formats: with every int8 product and norm replaced by its definition in 64 bits on
the same int8 rows, only roundings to bf16 differ (2^-8 each, a few dozen of them in random directions), so logits
agree to a cosine of 0.999.  Against the 16-bit model, an int8 value carries a uniform error of half a step, about
0.8 % of a normal row's standard deviation, in both operands of each product; eight products in two layers and the
exponentials of route and attention leave it below 10 %: cosine 0.99.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import double_attention_b200 as da
from double_attention_b200 import DoubleAttentionLM, eight_bit, experiment_config, int8_model, ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _cos(a: torch.Tensor, b: torch.Tensor) -> float:
    return F.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item()


def _lm(preset: str = "a1", layers: int = 2, **overrides) -> DoubleAttentionLM:
    torch.manual_seed(0)
    return DoubleAttentionLM(512, 160, experiment_config(preset, **overrides), layers, feedforward_dim=1536).cuda()


def _ids(batch: int, length: int) -> torch.Tensor:
    return torch.randint(0, 512, (batch, length), device="cuda", generator=torch.Generator("cuda").manual_seed(1))


def _plain_linear(x, weight, bias=None, *, gelu=False, dtype=BF16):
    y = (x.values.double() @ weight.values.double().t()) * x.scale.double()[..., None] * weight.scale.double()
    y = y if bias is None else y + bias.double()
    return (F.gelu(y) if gelu else y).to(dtype)


def _plain_quantize(y):
    amax = y.abs().amax(-1, keepdim=True)
    return da.Int8Rows((y / amax * 127).round().to(torch.int8), (amax[..., 0] / 127).float())


def _plain_norm(x, norm):
    return _plain_quantize(F.layer_norm(x.double(), x.shape[-1:], norm.weight.double(), norm.bias.double(), norm.eps))


@pytest.mark.parametrize(("preset", "length"), [("a1", 130), ("qk4-s4", 64), ("a1", 1)])
def test_int8_language_model(preset: str, length: int, monkeypatch) -> None:
    lm = _lm(preset).eval()
    ids = _ids(2, length)
    served = da.Int8DoubleAttentionLM(lm)
    logits = served(ids)
    assert logits.shape == (2, length, 512) and logits.dtype == BF16 and logits.isfinite().all()
    assert torch.equal(served(ids), logits)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        # (the 16-bit attention takes no fewer than 128 rows; later positions do not change earlier ones)
        full = lm(F.pad(ids, (0, max(0, 64 - length))))[0][:, :length]
    assert _cos(logits, full) >= 0.99
    monkeypatch.setattr(int8_model, "int8_linear", _plain_linear)
    monkeypatch.setattr(int8_model, "quantize_int8", lambda x: _plain_quantize(x.double()))
    monkeypatch.setattr(int8_model, "layernorm_int8", _plain_norm)
    monkeypatch.setattr(int8_model, "add_layernorm_int8", lambda x, b, n: (x + b, _plain_norm(x + b, n)))
    assert _cos(logits, served(ids)) >= 0.999
    ops.device_status()


def test_int8_language_model_weights_and_refusals() -> None:
    lm = _lm(layers=1)
    served = da.Int8DoubleAttentionLM(lm, torch.float16)
    assert served(_ids(1, 7)).dtype == torch.float16
    layer = served.blocks[0].first
    assert layer.weight.dtype == torch.int8 and layer.weight.shape == lm.stack.blocks[0].feedforward[0].weight.shape
    with pytest.raises(ValueError):
        served(_ids(1, 161))
    with pytest.raises(ValueError):
        served(_ids(1, 7)[0])
    with pytest.raises(ValueError):
        da.Int8DoubleAttentionLM(lm, torch.float32)
    with pytest.raises(RuntimeError):
        da.Int8DoubleAttentionLM(lm.cpu())


def test_language_model_trains_with_checkpoints_in_8_bits(monkeypatch) -> None:
    """One step with the feed-forward activations in 8 bits: the same loss (the forward does not change), gradients
    within what the checkpoints round, fewer bytes kept."""
    lm, ids = _lm(), _ids(4, 128)

    def step(kept: list):
        lm.zero_grad(set_to_none=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
            with torch.autocast("cuda", dtype=BF16):
                loss = lm(ids, ids.roll(-1, 1))[1]
        loss.backward()
        return loss.item(), {n: p.grad.clone() for n, p in lm.named_parameters() if p.grad is not None}

    monkeypatch.setattr(ops, "BLOCK_LINEAR_ON_TCGEN05", True)  # the forward that the checkpointed one equals
    full: list = []
    loss16, grads16 = step(full)
    monkeypatch.setattr(eight_bit, "FEEDFORWARD_CHECKPOINT8", True)
    kept: list = []
    loss8, grads8 = step(kept)
    assert loss8 == pytest.approx(loss16, rel=1e-4)
    assert set(grads8) == set(grads16)
    for name, g in grads16.items():
        assert _cos(grads8[name], g) >= 0.999, name
    rows, hidden, width = 4 * 128, 1536, 512
    saved = 2 * rows * (2 * width + 4 * hidden - (width + hidden) * 33 / 32)  # of x, z and h in 16 bits, two layers
    assert sum(full) - sum(kept) >= 0.9 * saved
    ops.device_status()
