"""The language model served in int8 as a module of its own: what it holds, and how it moves."""

from __future__ import annotations

import gc

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import DoubleAttentionLM, experiment_config

pytestmark = pytest.mark.gpu


def _lm(seed: int = 0, layers: int = 2, **overrides) -> DoubleAttentionLM:
    torch.manual_seed(seed)
    return DoubleAttentionLM(512, 160, experiment_config("a1", **overrides), layers, dictionary_group_size=1,
                             feedforward_dim=1536).cuda()


def _ids(*shape: int) -> torch.Tensor:
    return torch.randint(0, 512, shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))


def test_served_model_does_not_follow_the_trained_one() -> None:
    lm, ids = _lm(), _ids(2, 64)
    served = da.Int8DoubleAttentionLM(lm)
    logits = served(ids)
    before = {name: p.clone() for name, p in lm.named_parameters()}
    with torch.no_grad():
        for p in lm.parameters():
            p.mul_(1.25).add_(0.01)
    assert torch.equal(served(ids), logits)
    assert not torch.equal(da.Int8DoubleAttentionLM(lm)(ids), logits)
    with torch.no_grad():  # and the trained one is left as it is
        for p in served.parameters():
            p.zero_()
    assert all(torch.equal(p, 1.25 * before[name] + 0.01) for name, p in lm.named_parameters())
    assert all(p.requires_grad for p in lm.parameters()) and not any(p.requires_grad for p in served.parameters())


def test_state_dict_holds_all_of_the_served_model() -> None:
    served, other = da.Int8DoubleAttentionLM(_lm(0)), da.Int8DoubleAttentionLM(_lm(1))
    ids = _ids(2, 64)
    assert not torch.equal(other(ids), served(ids))
    other.load_state_dict(served.state_dict())
    assert torch.equal(other(ids), served(ids))


def test_served_model_moves_as_a_whole() -> None:
    ids = _ids(2, 64)
    da.Int8DoubleAttentionLM(_lm())(ids)  # (what the library itself keeps on the device is there from here on)
    gc.collect()
    before = torch.cuda.memory_allocated()
    served = da.Int8DoubleAttentionLM(_lm())
    logits = served(ids)
    served.to("cpu")
    gc.collect()
    assert {t.device.type for t in (*served.parameters(), *served.buffers())} == {"cpu"}
    assert torch.cuda.memory_allocated() - before <= logits.numel() * 2 + 1024, "tensors that no move reaches"
    assert torch.equal(served.to("cuda")(ids), logits)


@pytest.mark.parametrize("change", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(),
                                    lambda m: m.to("cpu", torch.float16).to("cuda"),
                                    lambda m: torch.nn.Sequential(m).half()[0]])
def test_types_stay_as_they_were_made(change) -> None:
    served, ids = da.Int8DoubleAttentionLM(_lm()), _ids(2, 64)
    logits, types = served(ids), {name: t.dtype for name, t in served.state_dict().items()}
    served = change(served)
    assert {name: t.dtype for name, t in served.state_dict().items()} == types
    assert torch.equal(served(ids), logits)
    torch.manual_seed(3)
    layer = da.Int8Linear(torch.randn(40, 200, device="cuda"), torch.randn(40, device="cuda"), torch.float16)
    x = torch.randn(5, 200, device="cuda")
    y = layer(x)
    assert torch.equal(change(layer)(x), y) and layer.scale.dtype == layer.bias.dtype == torch.float32


class _Adapted(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


@pytest.mark.parametrize("where", ["first", "second", "output", "lm_head"])
def test_layers_with_a_forward_of_their_own_are_refused(where: str) -> None:
    """Their weight alone would be served."""
    lm = _lm()
    block = lm.stack.blocks[1]
    old = {"first": block.feedforward[0], "second": block.feedforward[2], "output": block.attention.output,
           "lm_head": lm.lm_head}[where]
    for new in (_Adapted(old.in_features, old.out_features, old.bias is not None).cuda(), torch.nn.Sequential(old)):
        if where == "lm_head":
            lm.lm_head = new
        elif where == "output":
            block.attention.output = new
        else:
            block.feedforward[0 if where == "first" else 2] = new
        with pytest.raises(NotImplementedError, match="nn.Linear"):
            da.Int8DoubleAttentionLM(lm)


@pytest.mark.parametrize("shape", [(0, 5), (2, 0), (0, 0)])
def test_no_tokens_give_no_logits(shape: tuple[int, int]) -> None:
    for dtype in (torch.bfloat16, torch.float16):
        logits = da.Int8DoubleAttentionLM(_lm(layers=1), dtype)(_ids(*shape))
        assert logits.shape == (*shape, 512) and logits.dtype == dtype and logits.is_cuda
