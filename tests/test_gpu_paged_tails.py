"""Attention over a paged cache in fp16 where most of a row lies far below its largest weight.

Every sequence reads the same pages: one key whose score lies 17.5 nats above the others', whose weights are then
2^-25.2 of the largest, below half of fp16's smallest step.  There are as many sequences as the GPU has places for, so that
none is cut into pieces with offsets of their own.

Tolerances, fixed before the first run: as those of the other tests of these operators (each weight rounded to 16 bits,
eps / 2 of it, the result once; scores' drift 2 H R 2^-24 gamma |q| |k| + 1e-5 of A = sum softmax |V|), and for weights below
fp16's normal range half a step of 2^-24 each, 2^-25 against a largest weight of 2^7 or, where maps are mixed, 2^13: 2^-32 or
2^-38 a key of the largest |V|.
"""

from __future__ import annotations

import math

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import ops

pytestmark = pytest.mark.gpu
FP16 = torch.float16
EPS = torch.finfo(FP16).eps


def _run(sequences: int, new: int, length: int, maps: int, weights: list[float] | None, lift: int) -> None:
    g = torch.Generator("cuda").manual_seed(0)
    routing, dim, page, gamma, top = 64, 128, 64, 20.0, 5
    keys = torch.zeros(length, maps, routing, dtype=FP16, device="cuda")
    keys[:, :, 0] = 0.125              # a score of 2.5 everywhere,
    keys[top, 0, 0] = 1.0              # but 20 of map 0 at one position
    values = (0.5 + torch.rand(length, dim, device="cuda", generator=g)).to(FP16)
    values[top] = 0                    # what is left is the tail's
    query = torch.zeros(maps, sequences * new, routing, dtype=FP16, device="cuda")
    query[:, :, 0] = 1.0
    scales = torch.full((maps,), gamma, device="cuda")
    mix = None if weights is None else torch.tensor(weights, device="cuda")
    pages = length // page
    batch = da.PagedBatch(torch.arange(pages, dtype=torch.int32, device="cuda").repeat(sequences, 1),
                          torch.full((sequences,), length - new, dtype=torch.int32, device="cuda"),
                          torch.arange(sequences + 1, dtype=torch.int32, device="cuda") * new, new)
    y = da.routed_attention_paged(query, keys.view(pages, page, maps, routing), values.view(pages, page, dim), batch, scales, mix)
    want = 0
    hidden = torch.ones(new, length, dtype=torch.bool, device="cuda").triu(length - new + 1)
    for m in range(maps):
        score = (gamma * keys[None, :, m, 0].double()).expand(new, length).masked_fill(hidden, -math.inf)
        want = want + (1.0 if mix is None else mix[m].double()) * (torch.softmax(score, 1) @ values.double())
    bound = EPS * want + want * (2 * maps * routing * 2.0**-24 * gamma + 1e-5) + length * 2.0**-(25 + lift) * 1.5
    off = (y.view(sequences, new, dim).double() - want).abs()
    assert (off <= bound).all(), f"off by {(off / want).max().item():.2e} of the value, allowed {(bound / want).max().item():.2e}"
    assert ops.device_status() == 0


@pytest.mark.parametrize("new", [1, 3, 16])
def test_few_tokens_keep_a_far_tail(new) -> None:
    _run(300, new, 32768, 1, None, 7)


def test_chunks_keep_a_far_tail() -> None:
    _run(148, 20, 32768, 1, None, 7)


def test_chunks_keep_a_flat_map_beside_a_sharp_one() -> None:
    _run(74, 20, 131072, 2, [0.6, 0.4], 13)


def test_few_tokens_keep_a_flat_map_beside_a_sharp_one() -> None:
    _run(300, 2, 32768, 2, [0.6, 0.4], 7)
