"""The paged cache: appended keys and values, and the routed attention over the pages, against 64 bits.

Tolerances, fixed before the first run.  A call rounds every softmax weight to the pages' type before it multiplies the
values (eps / 2 of each weight), and its result once (eps / 2 of it).  Scores are fp32 sums of H R products: off by at most
H R 2^-24 |q| |k| gamma, which moves a weight by that share of itself and the row's sum by no more; exponentials, sums and
joins of fp32 partial results add less than 1e-5 of the weights.  With A = sum_s alpha_s softmax_s |V| the bound of every
element is  eps / 2 (A + |y|) + A (2 H R 2^-24 gamma |q| |k| + 1e-5).
"""

from __future__ import annotations

import math
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import ops, paged

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


class Case:
    """A cache whose unused slots hold ``fill``, sequences of ``held`` tokens and ``new`` more, all random."""

    def __init__(self, h, s, r, d, page, dtype, held, new, *, scale=16.0, norm=1.0, seed=0, behind=0, fill=math.nan):
        g = torch.Generator("cuda").manual_seed(seed)
        rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
        self.h, self.s, self.r, self.d, self.page, self.held, self.new = h, s, r, d, page, held, new
        need = [-(-(a + n) // page) for a, n in zip(held, new)]
        pages = sum(need) + 2
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((len(held), max(need + [1]) + 1), -7, dtype=torch.int32, device="cuda")  # past the need: anything
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        self.batch = da.PagedBatch(table, torch.tensor(held, dtype=torch.int32, device="cuda"), starts, max(new))
        n = sum(new) + behind
        unit = lambda t: (norm * t / t.norm(dim=-1, keepdim=True)).to(dtype)  # noqa: E731
        self.q, self.k = unit(rand(h, n, r)), unit(rand(h, n, r))
        self.v = rand(n, d).to(dtype)
        self.key_pages = torch.full((pages, page, h, r), fill, dtype=dtype, device="cuda")
        self.value_pages = torch.full((pages, page, d), fill, dtype=dtype, device="cuda")
        self.old = []
        for b, a in enumerate(held):
            k, v = unit(rand(a, h, r)), rand(a, d).to(dtype)
            self.old.append((k, v))
            slots = self.slots(b, range(a))
            self.key_pages.view(-1, h, r)[slots] = k
            self.value_pages.view(-1, d)[slots] = v
        self.scales = scale * (1 + 0.1 * torch.arange(s, device="cuda"))
        self.weights = torch.softmax(rand(s), 0) if s > 1 else None
        self.dtype, self.norm = dtype, norm

    def slots(self, b, positions):
        table = self.batch.table[b].tolist()
        return torch.tensor([table[j // self.page] * self.page + j % self.page for j in positions], dtype=torch.long, device="cuda")

    def append(self):
        da.append_paged(self.k, self.v, self.key_pages, self.value_pages, self.batch)

    def attend(self, weights="own", **kw):
        return da.routed_attention_paged(self.q, self.key_pages, self.value_pages, kw.pop("batch", self.batch), self.scales,
                                         self.weights if weights == "own" else weights, **kw)

    def expected(self, per_map=False):
        """``(y, bound)`` in 64 bits: [N, D], or [N, S, D]."""
        ys, bounds = [], []
        group = max(self.h // self.s, 1)
        for b, (ko, vo) in enumerate(self.old):
            first, n, a = sum(self.new[:b]), self.new[b], self.held[b]
            k = torch.cat((ko.double(), self.k[:, first:first + n].transpose(0, 1).double()))
            v = torch.cat((vo, self.v[first:first + n])).double()
            y, bound = [], []
            for i in range(self.s):
                hs = [i * group + e for e in range(group)] if self.h >= self.s else [i // (self.s // self.h)]
                score = sum(self.q[e, first:first + n].double() @ k[:, e].t() for e in hs) * self.scales[i].double() / group**0.5
                hidden = torch.ones(n, a + n, dtype=torch.bool, device="cuda").triu(a + 1)
                p = torch.softmax(score.masked_fill(hidden, -math.inf), 1)
                w = 1.0 if self.weights is None or per_map else self.weights[i].double()
                seen = torch.where(v.isfinite(), v, 0)  # (what is not is not seen, in the cases here)
                y.append(w * (p @ seen))
                bound.append(w * (p @ seen.abs()))
            if not n:
                continue
            y, big = (torch.stack(y, 1), torch.stack(bound, 1)) if per_map else (sum(y), sum(bound))
            eps = torch.finfo(self.dtype).eps
            drift = 2 * self.h * self.r * 2.0**-24 * self.scales.max().item() * self.norm**2 * 1.02 + 1e-5
            ys.append(y)
            bounds.append(eps / 2 * (big + y.abs()) + big * drift + 1e-12)
        return torch.cat(ys), torch.cat(bounds)

    def check(self, y, per_map=False):
        want, bound = self.expected(per_map)
        n = sum(self.new)
        far = (y[:n].double() - want).abs() - bound
        assert (far <= 0).all(), f"{int((far > 0).sum())} of {far.numel()} off, worst {far.max().item():.3e}"
        assert ops.device_status() == 0


# H, S, R, D, page
SHAPES = [(1, 1, 64, 128, 16), (1, 1, 256, 512, 64), (1, 1, 512, 512, 128), (2, 1, 256, 512, 32), (1, 2, 256, 256, 16),
          (2, 2, 128, 512, 64), (4, 4, 128, 512, 32), (4, 2, 64, 128, 16), (3, 3, 128, 256, 32), (1, 1, 192, 256, 16),
          (1, 4, 128, 512, 256)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_append_then_attend_a_ragged_batch(shape, dtype) -> None:
    case = Case(*shape, dtype, held=[0, 31, 500, 7, 64, 0], new=[1, 1, 3, 0, 17, 40])
    case.append()
    case.check(case.attend())


@pytest.mark.parametrize("shape", [(1, 1, 256, 512, 64), (4, 4, 128, 512, 16), (2, 2, 256, 128, 32)])
@pytest.mark.parametrize(("held", "new"), [([0], [1]), ([1], [1]), ([15], [1]), ([31], [1]), ([32], [1]), ([4095], [1]),
                                           ([20000], [1]), ([70, 20000, 3], [1, 1, 1]), ([3000] * 40, [1] * 40),
                                           ([0, 33], [33, 5]), ([1000], [64])])
def test_lengths_around_tiles_and_pages(shape, held, new) -> None:
    case = Case(*shape, BF16, held, new, seed=1)
    case.append()
    case.check(case.attend())


@pytest.mark.parametrize(("shape", "held", "new"), [((1, 1, 256, 512, 64), [0], [300]), ((1, 1, 512, 512, 128), [700], [129]),
                                                    ((4, 4, 128, 512, 32), [0, 900, 31], [256, 130, 1]),
                                                    ((1, 2, 256, 256, 16), [65, 0], [127, 128]),
                                                    ((2, 1, 128, 128, 64), [5000], [200]), ((1, 1, 64, 512, 16), [40], [1000]),
                                                    ((1, 1, 256, 512, 64), [3, 9000, 0, 700], [2, 65, 257, 1030]),
                                                    ((4, 4, 128, 512, 64), [2, 6000, 0, 700], [20, 65, 257, 630]),
                                                    ((3, 3, 128, 256, 128), [513], [300]), ((4, 2, 64, 128, 256), [513], [300]),
                                                    ((1, 1, 192, 256, 64), [513, 0], [300, 128]),
                                                    ((1, 1, 256, 512, 64), [300], [17]), ((4, 4, 128, 512, 64), [300, 0], [5, 6]),
                                                    ((2, 2, 128, 256, 16), [3000, 5], [9, 40]), ((1, 1, 512, 512, 64), [1000], [63])])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("fill", [math.nan, 30000.0])
def test_chunks(shape, held, new, dtype, fill) -> None:
    case = Case(*shape, dtype, held, new, seed=2, fill=fill)
    case.append()
    case.check(case.attend())
    case.check(case.attend(batch=case.batch._replace(max_new=None)))
    case.check(case.attend(batch=case.batch._replace(max_new=1)))  # a wrong guess changes no result


@pytest.mark.parametrize("new", [[1, 3], [200, 2]])
@pytest.mark.parametrize("shape", [(2, 2, 128, 256, 32), (4, 4, 128, 512, 64), (1, 3, 64, 128, 16)])
def test_outputs_of_each_map(shape, new) -> None:
    case = Case(*shape, BF16, [100, 2000], new, seed=3, fill=5.0)
    case.append()
    y = case.attend(weights=None)
    assert y.shape == (sum(new), case.s, case.d)
    case.check(y, per_map=True)


@pytest.mark.parametrize("new", [[2, 9], [150, 200]])
@pytest.mark.parametrize("norm", [30.0, 1e-3])
def test_scores_of_any_size(norm, new) -> None:
    """Sharp rows, whose largest score lies hundreds above the others, and flat ones."""
    for h, s in ((1, 1), (2, 2)):
        case = Case(h, s, 128, 256, 32, BF16, [600, 77], new, norm=norm, seed=4, scale=1.0 if norm > 1 else 16.0, fill=5.0)
        case.append()
        case.check(case.attend())


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_maximum_that_grows_along_the_keys(dtype) -> None:
    """Every key tile's scores lie far above the tile's before it, so that all earlier weights fade."""
    for h, s in ((1, 1), (2, 2)):
        case = Case(h, s, 128, 512, 64, dtype, [2500], [300], seed=15, fill=5.0)
        k, v = case.old[0]
        ramp = torch.linspace(0.05, 8.0, 2800, device="cuda")[:, None, None]
        direction = torch.nn.functional.normalize(torch.ones(128, device="cuda"), dim=0)
        noise = 0.02 * torch.randn(2800, h, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        keys = (ramp * direction + noise).to(dtype)
        case.old[0] = (keys[:2500], v)
        case.key_pages.view(-1, h, 128)[case.slots(0, range(2500))] = keys[:2500]
        case.k = keys[2500:].transpose(0, 1)
        case.q = (0.3 * case.q.float() + direction).to(dtype)
        case.norm = 8.5**0.5 * 1.4**0.5  # of the product |q| |k|
        case.append()
        case.check(case.attend())


@pytest.mark.parametrize("new", [[6, 40], [200, 170]])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_later_tokens_infinity_stays_out_of_earlier_rows(value, dtype, new) -> None:
    case = Case(2, 2, 128, 256, 32, dtype, [100, 30], new, seed=5)
    case.v[new[0] - 1] = value   # the first sequence's last new token
    case.v[sum(new) - 1, 3] = value
    case.append()
    y = case.attend()
    want, bound = case.expected()
    seen = torch.ones(sum(new), 256, dtype=torch.bool, device="cuda")
    seen[new[0] - 1] = False
    seen[sum(new) - 1, 3] = False
    assert ((y.double() - want).abs() <= bound)[seen].all()
    assert not y[~seen].isfinite().any()


@pytest.mark.parametrize("new", [[3, 0, 2], [140, 0, 131]])
def test_rows_behind_the_last_sequence(new) -> None:
    case = Case(1, 1, 128, 128, 16, BF16, [10, 20, 30], new, behind=11, seed=6)
    before = case.key_pages.clone(), case.value_pages.clone()
    case.append()
    written = torch.zeros(case.key_pages.shape[0] * 16, dtype=torch.bool, device="cuda")
    for b, (a, n) in enumerate(zip(case.held, case.new)):
        slots = case.slots(b, range(a, a + n))
        written[slots] = True
        first = sum(new[:b])
        assert torch.equal(case.key_pages.view(-1, 1, 128)[slots, 0], case.k[0, first:first + n])
        assert torch.equal(case.value_pages.view(-1, 128)[slots], case.v[first:first + n])
    for now, was in zip((case.key_pages, case.value_pages), before):
        assert torch.equal(now.view(torch.int16).flatten(0, 1)[~written], was.view(torch.int16).flatten(0, 1)[~written])
    y = case.attend()
    assert not y[sum(new):].any()
    case.check(y)
    out = torch.full_like(y, 5.0)
    assert case.attend(out=out) is out
    assert (out[sum(new):] == 5.0).all() and torch.equal(out[:sum(new)], y[:sum(new)])


@pytest.mark.parametrize("source", [torch.float32, BF16, FP16])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_append_converts_and_takes_any_strides(source, dtype) -> None:
    case = Case(2, 2, 64, 128, 16, dtype, [0, 20], [5, 30], seed=7)
    k = torch.randn(35, 2, 64 + 1, device="cuda").to(source)[..., 1:].transpose(0, 1)  # [H, N, R] off 16 bytes
    v = torch.randn(128, 35, device="cuda").to(source).t()
    da.append_paged(k, v, case.key_pages, case.value_pages, case.batch)
    for b, (a, n) in enumerate(zip(case.held, case.new)):
        slots, first = case.slots(b, range(a, a + n)), sum(case.new[:b])
        assert torch.equal(case.key_pages.view(-1, 2, 64)[slots], k.transpose(0, 1)[first:first + n].to(dtype))
        assert torch.equal(case.value_pages.view(-1, 128)[slots], v[first:first + n].to(dtype))


def test_query_and_table_of_other_strides() -> None:
    case = Case(2, 2, 128, 256, 32, BF16, [100, 300], [3, 20], seed=8)
    case.append()
    y = case.attend()
    wide = torch.randn(case.q.shape[1], 2, 200, device="cuda").to(BF16)
    wide[..., 8:136] = case.q.transpose(0, 1)
    table = torch.zeros(2, 40, dtype=torch.int32, device="cuda")
    table[:, :case.batch.table.shape[1]] = case.batch.table
    for q in (wide[..., 8:136].transpose(0, 1), wide[..., 8:136].contiguous().transpose(0, 1)):
        assert torch.equal(da.routed_attention_paged(q, case.key_pages, case.value_pages,
                                                     case.batch._replace(table=table[:, :case.batch.table.shape[1]]),
                                                     case.scales, case.weights), y)
    off = torch.zeros(case.q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(case.q)
    off.copy_(case.q)
    case.check(da.routed_attention_paged(off, case.key_pages, case.value_pages, case.batch, case.scales, case.weights))


@pytest.mark.parametrize("new", [[2, 3, 1], [140, 3, 150]])
@pytest.mark.parametrize("entry", [-1, 10**6])
def test_pages_outside_the_cache_are_reported_and_not_followed(entry, new) -> None:
    case = Case(1, 1, 128, 128, 16, BF16, [100, 300, 40], new, seed=9)
    case.append()
    want = case.attend()
    assert ops.device_status() == 0
    case.batch.table[1, 5] = entry
    y = case.attend()
    assert ops.device_status() == paged.BAD_PAGE
    rows = torch.zeros(sum(new), dtype=torch.bool, device="cuda")
    rows[new[0]:new[0] + new[1]] = True
    assert y[rows].isnan().all() and torch.equal(y[~rows], want[~rows])
    case.batch.table[1, 300 // 16] = entry
    before = case.key_pages.clone()
    case.append()
    assert ops.device_status() == paged.BAD_PAGE
    assert torch.equal(case.key_pages.view(torch.int16), before.view(torch.int16))  # (the others' were there already)


@pytest.mark.parametrize("new", [[2, 3], [150, 130]])
def test_lengths_that_the_table_cannot_hold(new) -> None:
    case = Case(1, 1, 128, 128, 16, BF16, [100, 40], new, seed=10)
    case.append()
    want = case.attend()
    for length in (10**9, -5, 2**31 - 1):
        lengths = case.batch.lengths.clone()
        lengths[0] = length
        y = case.attend(batch=case.batch._replace(lengths=lengths))
        assert ops.device_status() == paged.BAD_PAGE
        assert y[:new[0]].isnan().all() and torch.equal(y[new[0]:], want[new[0]:])
        da.append_paged(case.k, case.v, case.key_pages, case.value_pages, case.batch._replace(lengths=lengths))
        assert ops.device_status() == paged.BAD_PAGE


def test_on_another_stream_and_captured() -> None:
    case = Case(4, 4, 128, 512, 32, BF16, [1000, 40, 7], [1, 2, 160], seed=11)
    case.append()
    y = case.attend()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = case.attend()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, y)
    # a captured step follows the lengths and starts that it finds
    new_key, new_value = case.key_pages.clone(), case.value_pages.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        da.append_paged(case.k, case.v, new_key, new_value, case.batch)
        captured = da.routed_attention_paged(case.q, new_key, new_value, case.batch, case.scales, case.weights)
    graph.replay()
    assert torch.equal(captured, y)
    case.batch.lengths.sub_(torch.tensor([10, 3, 7], dtype=torch.int32, device="cuda"))
    graph.replay()
    moved = da.routed_attention_paged(case.q, new_key, new_value, case.batch, case.scales, case.weights)
    assert torch.equal(captured, moved) and not torch.equal(moved, y)
    assert ops.device_status() == 0


def test_no_tokens_and_no_sequences() -> None:
    case = Case(1, 1, 128, 128, 16, BF16, [100, 40], [2, 3], seed=12)
    none = torch.zeros_like(case.batch.starts)
    y = case.attend(batch=case.batch._replace(starts=none))
    assert not y.any()
    empty = da.PagedBatch(case.batch.table[:0], case.batch.lengths[:0], none[:1], 0)
    assert not case.attend(batch=empty).any()
    da.append_paged(case.k, case.v, case.key_pages, case.value_pages, empty)
    y = da.routed_attention_paged(case.q[:, :0], case.key_pages, case.value_pages, case.batch._replace(starts=none), case.scales)
    assert y.shape == (0, 128)
    assert ops.device_status() == 0


@pytest.mark.parametrize("new", [[3, 20], [150, 200]])
@pytest.mark.parametrize("weights", [[0.0, 1.0], [-0.5, 1.5], [0.0, 0.0], [1e-6, 2.0]])
def test_map_weights_of_any_sign(weights, new) -> None:
    case = Case(2, 2, 128, 256, 32, BF16, [100, 300], new, seed=17, fill=5.0)
    case.append()
    case.weights = torch.tensor(weights, device="cuda")
    want, _ = case.expected()
    per_map, each = case.expected(per_map=True)
    # (each map's bound counts by its weight; the mixture is rounded once)
    bound = (each * case.weights.abs()[:, None].double()).sum(1) + torch.finfo(BF16).eps / 2 * want.abs() + 1e-12
    assert ((case.attend().double() - want).abs() <= bound).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("new", [[3, 20], [150, 200]])
@pytest.mark.parametrize("scale", [0.0, -16.0, 200.0])
def test_temperatures_of_any_sign(scale, new) -> None:
    for h, s in ((1, 1), (4, 4)):
        case = Case(h, s, 128, 256, 32, FP16, [100, 700], new, scale=scale, seed=18, fill=5.0)
        case.append()
        want, bound = case.expected()
        if scale < 0:
            bound = bound + 2 * 2 * h * 128 * 2.0**-24 * 16 * 1.3 * want.abs().max()  # (expected() counts the drift of gamma, not |gamma|)
        assert ((case.attend().double() - want).abs() <= bound).all()


def test_starts_that_leave_rows_out_or_do_not_rise() -> None:
    case = Case(1, 1, 128, 128, 16, BF16, [100, 300, 40], [70, 80, 90], seed=19, fill=5.0)
    case.append()
    starts = case.batch.starts.clone()
    starts[0] = 66  # rows 0 to 65 belong to no sequence; the first one's four rows are its first four
    y = case.attend(batch=case.batch._replace(starts=starts))
    assert not y[:66].any() and torch.equal(y[70:], case.attend()[70:])
    # sequences that overlap, more tokens than rows: nothing outside is touched, and nothing is waited for
    table, lengths = case.batch.table[:1].repeat(64, 1), torch.zeros(64, dtype=torch.int32, device="cuda")
    falling = torch.tensor([0, 240] * 32 + [0], dtype=torch.int32, device="cuda")
    around = torch.full((242, 128), 7.0, dtype=BF16, device="cuda")
    case.attend(batch=da.PagedBatch(table, lengths, falling), out=around[1:241])
    assert (around[0] == 7.0).all() and (around[241] == 7.0).all()
    ops.device_status()


def test_one_token_of_any_strides() -> None:
    case = Case(2, 2, 128, 256, 32, BF16, [100], [1], seed=20)
    case.append()
    odd = torch.as_strided(case.q.transpose(0, 1).contiguous(), (2, 1, 128), (128, 3, 1))
    assert torch.equal(da.routed_attention_paged(odd, case.key_pages, case.value_pages, case.batch, case.scales, case.weights),
                       case.attend())


def test_many_sequences() -> None:
    held, new = [b * 37 % 200 for b in range(700)], [b % 3 for b in range(700)]
    case = Case(1, 1, 64, 128, 16, BF16, held, new, seed=13)
    case.append()
    case.check(case.attend())


def test_a_long_cache_past_32_bits_of_elements() -> None:
    """The last pages of a cache whose values have more than 2^31 elements."""
    h, r, d, page, pages = 1, 64, 512, 64, 70000
    assert pages * page * d > 2**31
    keys = torch.zeros(pages, page, h, r, dtype=BF16, device="cuda")
    values = torch.zeros(pages, page, d, dtype=BF16, device="cuda")
    n, held = 5, 300
    table = torch.arange(pages - 1, pages - 7, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(0)
    q, k = (torch.nn.functional.normalize(torch.randn(1, held + n, r, device="cuda", generator=g), dim=-1).to(BF16) for _ in range(2))
    v = torch.randn(held + n, d, device="cuda", generator=g).to(BF16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    da.append_paged(k[:, :held], v[:held], keys, values, da.PagedBatch(table, zero, torch.tensor([0, held], dtype=torch.int32, device="cuda")))
    batch = da.PagedBatch(table, zero + held, starts, n)
    da.append_paged(k[:, held:], v[held:], keys, values, batch)
    scales = torch.tensor([16.0], device="cuda")
    y = da.routed_attention_paged(q[:, held:], keys, values, batch, scales)
    score = (q[0, held:].double() @ k[0].double().t() * 16).masked_fill(
        torch.ones(n, held + n, dtype=torch.bool, device="cuda").triu(held + 1), -math.inf)
    p = torch.softmax(score, 1)
    big = p @ v.double().abs()
    bound = 2**-8 * (big + (p @ v.double()).abs()) + big * (2 * r * 2.0**-24 * 16 * 1.02 + 1e-5)
    assert ((y.double() - p @ v.double()).abs() <= bound).all()
    assert ops.device_status() == 0


_ALONE = """
import sys
sys.path.insert(0, {tests!r})
from test_gpu_paged import BF16, FP16, Case
for shape in [(1, 1, 256, 512, 64), (4, 4, 128, 512, 64), (3, 3, 128, 256, 32), (2, 2, 256, 512, 16), (4, 2, 64, 128, 128)]:
    for held, new in (([4000, 300], [500, 129]), ([0], [640]), ([20000], [65])):
        case = Case(*shape, FP16, held, new, fill=5.0, seed=16)
        case.append()
        for _ in range(3):
            case.check(case.attend())
print("alone: ok")
"""


def test_kernels_one_after_another() -> None:
    """Each kernel alone on the GPU (launches that block), so that none finds its input's producer still running."""
    done = subprocess.run([sys.executable, "-c", _ALONE.format(tests=str(Path(__file__).parent))], capture_output=True, text=True,
                          timeout=300, env=os.environ | {"CUDA_LAUNCH_BLOCKING": "1"}, cwd=Path(__file__).parent.parent)
    assert done.returncode == 0 and "alone: ok" in done.stdout, done.stdout[-2000:] + done.stderr[-2000:]


def test_refusals() -> None:
    case = Case(2, 2, 128, 256, 32, BF16, [10], [2], seed=14)
    args = (case.q, case.key_pages, case.value_pages, case.batch, case.scales, case.weights)

    def call(**change):
        named = dict(zip(("query", "key_pages", "value_pages", "batch", "scales", "map_weights"), args)) | change
        return da.routed_attention_paged(**named)

    with pytest.raises(ValueError, match="int32"):
        call(batch=case.batch._replace(lengths=case.batch.lengths.long()))
    with pytest.raises(ValueError, match="starts"):
        call(batch=case.batch._replace(starts=case.batch.starts[:1]))
    with pytest.raises(ValueError, match="type"):
        call(query=case.q.half())
    with pytest.raises(ValueError, match="query"):
        call(query=case.q[:1])
    with pytest.raises(ValueError, match="power of two"):
        call(key_pages=case.key_pages[:, :24].contiguous(), value_pages=case.value_pages[:, :24].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        call(value_pages=case.value_pages[..., ::2])
    with pytest.raises(ValueError, match="map weights"):
        call(map_weights=case.weights[:1])
    with pytest.raises(ValueError, match="one scale a map"):
        call(scales=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="one device"):
        call(scales=case.scales.cpu())
    with pytest.raises(ValueError, match="writes"):
        call(out=torch.empty(2, 256, device="cuda"))
    with pytest.raises(RuntimeError, match="no backward"):
        call(query=case.q.clone().requires_grad_())
    with pytest.raises(NotImplementedError):
        call(value_pages=case.value_pages[..., :64].contiguous())
    with pytest.raises(ValueError, match="keys"):
        da.append_paged(case.k[:, :1], case.v, case.key_pages, case.value_pages, case.batch)
    with pytest.raises(ValueError, match="float32"):
        da.append_paged(case.k.double(), case.v, case.key_pages, case.value_pages, case.batch)
    with pytest.raises(RuntimeError, match="no backward"):
        da.append_paged(case.k, case.v.clone().requires_grad_(), case.key_pages, case.value_pages, case.batch)
    assert ops.device_status() == 0


@pytest.mark.parametrize(("dims", "held", "new"), [((2, 1, 256, 256, 16), [1099] * 9, [176] * 9), ((1, 1, 256, 512, 64), [9000], [300]),
                                                   ((2, 1, 256, 512, 32), [30000], [73])])
def test_a_maximum_that_grows_at_any_tile(dims, held, new) -> None:
    """Scores so far apart that rows' maxima grow by much at late tiles too, whose products the two groups wait for."""
    case = Case(*dims, BF16, held, new, scale=1000.0)
    case.append()
    for _ in range(3):
        case.check(case.attend())
