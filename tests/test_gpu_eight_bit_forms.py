"""The eight-bit operators' kernel forms that need their own sizes or types, against the definition in 64 bits: norms of
every pair of residual and branch types, weight gradients with several accumulator chunks and several tiles for
each pair of CTAs, dense checkpoints that run over many blocks of threads.

Tolerances, fixed from the formulas before their first run: an int8 row is within half a step of the exact value,
plus the fp32 error of the row's factors (below 2e-3 steps).  A weight gradient's accumulator takes 64 instructions of 16 rows
before its sum moves on; each may cut the sum so far by one last place, 2^-23 of it at most and 0.72 * 2^-24 = 4.3e-8 on
average.  With all terms positive the sum grows evenly, so the cuts of a chunk are at most 2^-23 * (1 + ... + 64) / 64 =
32.5 * 2^-23 of it, 1.4e-6 on average; every addition of a chunk's or a split's sum rounds by 2^-24 of the total, up or
down.  One chain over all rows that cut so, computed in that way on the CPU, comes out 2.5e-5 low at 20481 rows
and 8e-5 at 66561, which the first bound refuses; over a split's 3392 rows 2.2e-6 to 5e-6 low in every element, which
the bound of the mean refuses.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import double_attention_b200 as da
from double_attention_b200 import ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUNDING = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}     # unit roundoff 2^-p of 24, 8 and 11 significant bits
SMALLEST = {F32: 2.0**-150, BF16: 2.0**-134, F16: 2.0**-25}  # half the smallest subnormal
CDF = 4e-7  # GELU's distribution function: its polynomial's 1.4e-7 and a few fp32 roundings


def _randn(*shape: int, seed: int = 0, dtype=F32) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.fixture(autouse=True)
def _no_grad_and_clean_status():
    with torch.no_grad():
        yield
    torch.cuda.synchronize()
    assert ops.device_status() == 0


# ----------------------------------------------------------------------------- norms
def _norm(kind: str, d: int, dtype):
    norm = (nn.RMSNorm if kind == "rms" else nn.LayerNorm)(d, eps=1e-6).cuda().to(dtype).requires_grad_(False)
    norm.weight.copy_(1 + 0.3 * _randn(d, seed=3))
    if kind == "layer":
        norm.bias.copy_(0.2 * _randn(d, seed=4))
    return norm


def _norm64(r: torch.Tensor, norm) -> torch.Tensor:
    r = r.double()
    if isinstance(norm, nn.LayerNorm):
        r = r - r.mean(-1, keepdim=True)
    y = r / torch.sqrt(r.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
    return y + norm.bias.double() if isinstance(norm, nn.LayerNorm) else y


def _check_int8(rows: da.Int8Rows, y: torch.Tensor) -> None:
    step = y.abs().amax(-1, keepdim=True) / 127
    got = rows.values.double() * rows.scale.double()[..., None]
    assert (got - y).abs().le(0.502 * step).all()
    assert (rows.scale.double() - step[..., 0]).abs().le(1e-5 * step[..., 0]).all()


# a warp a row; 64, 128 and 256 threads a row; a number of threads that the kernel is told; each on 16-byte rows and not
@pytest.mark.parametrize("d", [512, 501, 2048, 1999, 4000, 4001, 8192, 7997, 5000, 5003])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norms_of_every_residual_with_every_branch(kind: str, d: int) -> None:
    add = da.add_rmsnorm_int8 if kind == "rms" else da.add_layernorm_int8
    for dtype in (F32, BF16, F16):
        for branch_dtype in (F32, BF16, F16):
            for weight_dtype in {F32, dtype}:
                norm = _norm(kind, d, weight_dtype)
                x, branch = (2 * _randn(21, d, seed=d) + 0.5).to(dtype), _randn(21, d, seed=d + 1, dtype=branch_dtype)
                x_out, rows = add(x, branch, norm)
                assert torch.equal(x_out, (x.float() + branch.float()).to(dtype))
                _check_int8(rows, _norm64(x_out, norm))


def test_broadcast_rows_equal_the_row_alone() -> None:
    for d in (40, 501, 9000):
        x = _randn(6, d, seed=1)
        alone, same = da.quantize_int8(x[:1]), da.quantize_int8(x[:1].expand(5, d))
        assert torch.equal(same.values, alone.values.expand(5, d)) and torch.equal(same.scale, alone.scale.expand(5))


# ----------------------------------------------------------------------------- weight gradient
# (rows, N, K): q turned into X in the kernel up to 768 columns of dY, in memory first above.  More tiles than pairs of
# CTAs (a pair's second tile starts at a later stage, chunk and parity than its first); many chunks an item, alone
# and in splits; a last chunk of one ragged stage.
WGRAD = [(5000, 768, 6600), (5000, 2304, 2304), (1000, 700, 6900), (60_000, 512, 512), (40_001, 1024, 256), (66_561, 2304, 2304),
         (20_481, 768, 6400)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "n", "k"), WGRAD)
def test_weight_grad_of_many_chunks_and_items(rows: int, n: int, k: int, dtype) -> None:
    # magnitudes from 1/2 to 3/2, so that every term counts; first all positive (a sum of both signs is at most as long
    # as that of its magnitudes, so the bound holds for it too), then of both signs
    x = (0.5 + torch.rand(rows, k, generator=torch.Generator("cuda").manual_seed(1), device="cuda")).to(dtype)
    dy = (0.5 + torch.rand(rows, n, generator=torch.Generator("cuda").manual_seed(2), device="cuda")).to(dtype)
    kept = da.checkpoint8(x)
    positive = kept.restore()
    size = dy.double().t() @ positive.double()
    adds = -(-rows // 1024) + 74  # of chunks and of splits
    allowed = (32.5 * 2.0**-23 + adds * 2.0**-24) * size
    dw = da.weight_grad_checkpoint8(dy, kept, F32)
    assert (dw.double() - size).abs().le(allowed).all()
    assert ((dw.double() - size) / size).mean().abs() <= 2e-6
    # a sign for each row and for each column: sums stay near the square root of their length
    flip = lambda size, seed: torch.randint(0, 2, size, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * 2 - 1
    dy.mul_(flip((rows, 1), 3))
    x.mul_(flip((1, k), 4))
    kept = da.checkpoint8(x)
    want = dy.double().t() @ kept.restore().double()
    for out in (F32, dtype):
        dw = da.weight_grad_checkpoint8(dy, kept, out)
        assert (dw.double() - want).abs().le(allowed + 1.01 * ROUNDING[out] * want.abs() + SMALLEST[out]).all()
        assert torch.equal(dw, da.weight_grad_checkpoint8(dy, kept, out)), "two runs differ"


# ----------------------------------------------------------------------------- checkpoints
def _kept64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Values and exponents by the definition (finite values)."""
    low, high = (-24, 9) if x.dtype == F16 else (-126, 121)
    d = x.shape[-1]
    v = F.pad(x.double(), (0, -d % 32)).unflatten(1, (-1, 32))
    a = v.abs().amax(2, keepdim=True)
    e = torch.full_like(a, high)
    for candidate in range(high, low - 1, -1):
        e = torch.where(a <= 127 * 2.0**candidate, torch.full_like(e, candidate), e)
    q = (v / torch.exp2(e)).round().clamp(-127, 127)
    return q.flatten(1).to(torch.int8), e[..., 0].to(torch.int8)


def _gelu64(z: torch.Tensor) -> torch.Tensor:
    return z * torch.special.ndtr(z)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "d"), [(700, 1001), (3000, 33), (5001, 31), (40_000, 1), (9, 9001), (300, 1000)])
def test_dense_checkpoints_of_many_blocks(rows: int, d: int, dtype) -> None:
    size = torch.exp2((_randn(rows, 1, seed=9) * 3).clamp(-9, 9))  # rows of different exponents
    z, dh = (2.5 * size * _randn(rows, d, seed=d)).to(dtype), _randn(rows, d, seed=d + 1, dtype=dtype)
    q, e = _kept64(z)
    plain = da.checkpoint8(z)
    h, kept = da.gelu_checkpoint8(z)
    for c in (plain, kept):
        assert torch.equal(c.values, q) and torch.equal(c.exponent, e)
    want = _gelu64(z.double())
    assert (h.double() - want).abs().le(1.01 * ROUNDING[dtype] * want.abs() + CDF * z.double().abs() + SMALLEST[dtype]).all()
    zk = (q.double() * torch.exp2(e.double()).repeat_interleave(32, 1))[:, :d]
    assert torch.equal(kept.restore().double(), zk)
    dz, again = da.gelu_checkpoint8_backward(dh, kept)
    slope = torch.special.ndtr(zk) + zk * torch.exp(-zk * zk / 2) * 0.3989422804014327
    want = dh.double() * slope
    assert (dz.double() - want).abs().le(1.01 * ROUNDING[dtype] * want.abs()
                                         + 2 * CDF * (1 + zk.abs()) * dh.double().abs() + SMALLEST[dtype]).all()
    want = _gelu64(zk)
    assert (again.double() - want).abs().le(1.01 * ROUNDING[dtype] * want.abs() + CDF * zk.abs() + SMALLEST[dtype]).all()
    # rows on 16-byte words, which take another form, give the same bits
    wide = -d % 8 + 8
    h1, kept1 = da.gelu_checkpoint8(F.pad(z, (0, wide))[:, :d])
    dz1, again1 = da.gelu_checkpoint8_backward(F.pad(dh, (0, wide))[:, :d], kept)
    assert torch.equal(h1, h) and torch.equal(kept1.values, q) and torch.equal(kept1.exponent, e)
    assert torch.equal(dz1, dz) and torch.equal(again1, again)
