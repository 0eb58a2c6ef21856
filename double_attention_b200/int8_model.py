"""A trained ``DoubleAttentionLM`` served in int8.

:class:`Int8DoubleAttentionLM` quantises every Linear of the model once (a scale per output channel) and runs
its forward on the eight-bit operators: each norm adds the pending branch and leaves int8 rows, the projections
and the feed-forward layers multiply int8 rows, the route and the outer attention between them stay on their
16-bit kernels.  Per layer that is five int8 products (Q and K together, V, output, two of the feed-forward)
between two fused norms.  Inference only; the model it is built from is left as it is, and nothing that happens to it
later reaches the served one.

Measured, 6 layers of a1, feed-forward 1536, vocabulary 2048 (the 16-bit model under autocast beside it): 16 x 1024
tokens in 1.44 ms (2.39), replayed from a CUDA graph 1.34 (1.62); 64 x 1024 4.65 (5.89); 1 x 128 0.82 (2.38), from a graph
0.44 (0.48); a single token 1.0, from a graph 0.32.
"""

from __future__ import annotations

import copy

import torch
from torch import Tensor, nn

from . import ops
from .eight_bit import Int8Rows, add_layernorm_int8, int8_linear, layernorm_int8, own_forward, quantize_int8
from .modules import DoubleAttentionBlock, DoubleAttentionLM

_HALF = (torch.float16, torch.bfloat16)
_ATTENTION_ROWS = 128  # rows (batch times length) below which the attention kernels have no tile


class _FixedTypes(nn.Module):
    """A module that moves between devices and keeps its tensors' types: ``half()``, ``to(dtype)`` and the like on it
    or on a module around it leave them, since its products read int8 values with fp32 scales."""

    def _apply(self, fn, recurse: bool = True):
        def move(t: Tensor) -> Tensor:
            moved = fn(t)
            return moved if moved.dtype == t.dtype else t.to(moved.device)

        return super()._apply(move, recurse)


class Int8Linear(_FixedTypes):
    """A Linear whose weight is held in int8 with a scale per output channel and whose bias in fp32.

    ``forward`` takes int8 rows, or activations that it quantises per token first; with ``gelu`` the output
    goes through GELU in the product's epilogue.  ``dtype`` is the output's; ``half()`` and ``to(dtype)`` change no type."""

    def __init__(self, weight: Tensor, bias: Tensor | None, dtype: torch.dtype) -> None:
        super().__init__()
        rows = quantize_int8(weight.detach())
        self.register_buffer("weight", rows.values)
        self.register_buffer("scale", rows.scale)
        self.register_buffer("bias", None if bias is None else bias.detach().float().clone())
        self.dtype = dtype

    def forward(self, x: Tensor | Int8Rows, *, gelu: bool = False) -> Tensor:
        rows = x if isinstance(x, Int8Rows) else quantize_int8(x)
        return int8_linear(rows, Int8Rows(self.weight, self.scale), self.bias, gelu=gelu, dtype=self.dtype)


def _int8(layer: nn.Module, dtype: torch.dtype) -> Int8Linear:
    if own_forward(layer, nn.Linear):
        raise NotImplementedError(f"int8 serving covers layers that compute as nn.Linear does, got {layer}")
    return Int8Linear(layer.weight, layer.bias, dtype)


def _frozen(module: nn.Module) -> nn.Module:
    return copy.deepcopy(module).requires_grad_(False)


class _Bank(nn.Module):
    """A bank's normalised dictionaries as the route reads them."""

    def __init__(self, views: ops.DictionaryViews) -> None:
        super().__init__()
        for name in ("key", "key_t", "value", "value_t", "key_max"):
            self.register_buffer(name, getattr(views, name).clone())

    def views(self) -> ops.DictionaryViews:
        return ops.DictionaryViews(self.key, self.key_t, self.value, self.value_t, self.key_max, self.key, self.value)


class _Int8Block(nn.Module):
    def __init__(self, block: DoubleAttentionBlock, dtype: torch.dtype) -> None:
        super().__init__()
        attention, cfg = block.attention, block.attention.config
        if cfg.q_dictionary_feedforward:
            raise NotImplementedError("int8 serving does not cover the Q-dictionary feed-forward")
        first, act, second, _ = block.feedforward
        if own_forward(act, nn.GELU) or act.approximate != "none":
            raise NotImplementedError(f"int8 serving covers the exact form of GELU, got {act}")
        self.config = cfg
        self.attention_norm, self.feedforward_norm = _frozen(block.attention_norm), _frozen(block.feedforward_norm)
        self.query_key = Int8Linear(torch.cat((attention.query.weight, attention.key.weight)), None, dtype)
        self.value = Int8Linear(attention.value.weight, attention.value.bias, torch.bfloat16)  # as the attention reads it
        self.output = None if type(attention.output) is nn.Identity else _int8(attention.output, dtype)
        self.first, self.second = _int8(first, dtype), _int8(second, dtype)
        beta, scales = ops.temperatures(attention.log_beta, attention.log_score_scales)
        self.register_buffer("beta", beta.clone())
        self.register_buffer("scales", scales.clone())
        logits = attention.map_mix_logits
        self.register_buffer("map_weights", None if logits is None else torch.softmax(logits.float(), dim=0))

    def attend(self, rows: Int8Rows, views: ops.DictionaryViews) -> Tensor:
        cfg = self.config
        batch, tokens = rows.scale.shape
        projected, value = self.query_key(rows), self.value(rows)
        length = tokens
        if cfg.causal and batch * tokens < _ATTENTION_ROWS:
            # positions after the last one, which no query sees, fill the attention's smallest tile
            length = -(-_ATTENTION_ROWS // batch)
            projected = nn.functional.pad(projected, (0, 0, 0, length - tokens))
            value = nn.functional.pad(value, (0, 0, 0, length - tokens))
        routed = ops.route_projected(projected.view(batch * length, -1), views, self.beta, cfg, batch, length)
        if cfg.map_combine == "weighted_sum":
            combined = ops.routed_attention_mixed(routed, value, self.scales, self.map_weights, cfg)
        else:
            combined = ops.routed_attention_maps(routed, value, self.scales, cfg).permute(0, 2, 1, 3).flatten(2)
        combined = combined[:, :tokens]
        return combined if self.output is None else self.output(combined)

    def forward(self, x: Tensor, pending: Tensor | None, views: ops.DictionaryViews) -> tuple[Tensor, Tensor]:
        """``x + pending`` through the block; returns the residual and the feed-forward branch still to be added."""
        if pending is None:
            rows = layernorm_int8(x, self.attention_norm)
        else:
            x, rows = add_layernorm_int8(x, pending, self.attention_norm)
        x, rows = add_layernorm_int8(x, self.attend(rows, views), self.feedforward_norm)
        return x, self.second(self.first(rows, gelu=True))


class Int8DoubleAttentionLM(_FixedTypes):
    """``DoubleAttentionLM`` in int8: ``Int8DoubleAttentionLM(lm)(token_ids)`` gives the logits [B, T, V].

    ``lm`` must be on an sm_100 GPU.  What it has learned is copied, all at this moment: a later training step or
    ``load_state_dict`` of ``lm`` changes nothing here, and all of it is in this module's ``state_dict``.  Hooks
    on ``lm``'s modules do not run here; layers with a forward of their own are refused.  ``dtype`` is
    the 16-bit type of the activations between the int8 products and of the logits; no type changes later."""

    def __init__(self, lm: DoubleAttentionLM, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        if dtype not in _HALF:
            raise ValueError(f"int8 serving computes in bfloat16 or float16 between its products, got {dtype}")
        weight = lm.token_embedding.weight
        ops.resolve_backend("auto", weight, dtype)
        with torch.no_grad():
            self.max_sequence_length = lm.max_sequence_length
            self.token_embedding, self.position_embedding = _frozen(lm.token_embedding), _frozen(lm.position_embedding)
            self.final_norm = _frozen(lm.final_norm)
            stack = lm.stack
            self.blocks = nn.ModuleList(_Int8Block(b, dtype) for b in stack.blocks)
            self.lm_head = _int8(lm.lm_head, dtype)
            self.banks = nn.ModuleList(_Bank(ops.dictionary_views(b.raw_key, b.raw_value, stack.config.eps, dtype))
                                       for b in stack.banks)
            self._bank_of = [min(i // stack.dictionary_group_size, len(stack.banks) - 1) for i in range(len(stack.blocks))]

    @torch.no_grad()
    def forward(self, token_ids: Tensor) -> Tensor:
        if token_ids.ndim != 2:
            raise ValueError("token_ids must have shape [B, T]")
        length = token_ids.shape[1]
        if length > self.max_sequence_length:
            raise ValueError(f"sequence length {length} exceeds configured maximum {self.max_sequence_length}")
        if not token_ids.numel():
            return self.token_embedding.weight.new_empty(*token_ids.shape, self.lm_head.weight.shape[0], dtype=self.lm_head.dtype)
        positions = torch.arange(length, device=token_ids.device)
        x = (self.token_embedding(token_ids) + self.position_embedding(positions)[None]).float()
        views = [bank.views() for bank in self.banks]
        pending = None
        for block, bank in zip(self.blocks, self._bank_of):
            x, pending = block(x, pending, views[bank])
        return self.lm_head(add_layernorm_int8(x, pending, self.final_norm)[1])
