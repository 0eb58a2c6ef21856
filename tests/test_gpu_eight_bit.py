"""The eight-bit operators against their definitions in 64 bits.

Tolerances, fixed from the formulas: an int8 row is within half a step of the exact value (plus the fp32
error of the row's factors, below 2e-3 steps); an int8 product is exact before its scaling, so only the
four fp32 roundings behind it and the output's own rounding remain; GELU's distribution function carries
its polynomial's 1.4e-7 and a few fp32 roundings, below 4e-7; a checkpoint's values are exact.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import double_attention_b200 as da
from double_attention_b200 import eight_bit, ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUNDING = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}   # unit roundoff 2^-p of 24, 8 and 11 significant bits
SMALLEST = {F32: 2.0**-150, BF16: 2.0**-134, F16: 2.0**-25}  # half the smallest subnormal
CDF = 4e-7


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape: int, seed: int = 0, dtype=F32) -> torch.Tensor:
    return torch.randn(*shape, generator=_gen(seed), device="cuda").to(dtype)


@pytest.fixture(autouse=True)
def _no_grad_and_clean_status():
    with torch.no_grad():
        yield
    torch.cuda.synchronize()
    assert ops.device_status() == 0


# ----------------------------------------------------------------------------- norms and the row quantiser
def _norm64(r: torch.Tensor, kind: str, weight, bias, eps: float) -> torch.Tensor:
    r = r.double()
    if kind == "quantize":
        return r
    if kind == "layer":
        r = r - r.mean(-1, keepdim=True)
    y = r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def _check_int8(rows: da.Int8Rows, y: torch.Tensor) -> None:
    assert rows.values.shape == y.shape and rows.scale.shape == y.shape[:-1]
    step = y.abs().amax(-1, keepdim=True) / 127
    got = rows.values.double() * rows.scale.double()[..., None]
    assert (got - y).abs().le(0.502 * step).all()
    assert (rows.scale.double() - step[..., 0]).abs().le(1e-5 * step[..., 0]).all()
    live = step[..., 0] > 0
    assert rows.values.abs().amax(-1)[live].eq(127).all()


def _norm(kind: str, d: int, dtype=F32, affine: bool = True):
    norm = (nn.RMSNorm if kind == "rms" else nn.LayerNorm)(d, eps=1e-6, elementwise_affine=affine).cuda().to(dtype)
    if affine:
        norm.weight.copy_(1 + 0.3 * _randn(d, seed=3))
        if kind == "layer":
            norm.bias.copy_(0.2 * _randn(d, seed=4))
    return norm.requires_grad_(False)


NORM_SHAPES = [(1, 1), (1, 512), (5, 3), (37, 64), (129, 512), (64, 1000), (33, 1001), (17, 1024), (9, 1032), (7, 2500),
               (5, 4097), (3, 8192), (3, 10000), (2, 32768), (2, 32775), (2, 40000)]


@pytest.mark.parametrize("kind", ["rms", "layer", "quantize"])
@pytest.mark.parametrize(("rows", "d"), NORM_SHAPES)
def test_int8_rows_match_their_definition(kind: str, rows: int, d: int) -> None:
    for i, dtype in enumerate((F32, BF16, F16)):
        x = (2 * _randn(rows, d, seed=d + i) + (0.5 if d > 1 else 3.0)).to(dtype)
        if kind == "quantize":
            _check_int8(da.quantize_int8(x), x.double())
            continue
        if kind == "layer" and d == 1:
            continue  # a single column has no variance: its LayerNorm is the bias alone
        norm = _norm(kind, d, dtype=(F32, F32, BF16)[i])
        plain = (da.rmsnorm_int8 if kind == "rms" else da.layernorm_int8)(x, norm)
        weight, bias = norm.weight, getattr(norm, "bias", None)
        _check_int8(plain, _norm64(x, kind, weight, bias, 1e-6))
        branch = _randn(rows, d, seed=d + 7, dtype=(BF16, F16, F32)[i])
        add = da.add_rmsnorm_int8 if kind == "rms" else da.add_layernorm_int8
        x_out, both = add(x, branch, norm)
        assert torch.equal(x_out, (x.float() + branch.float()).to(dtype))
        _check_int8(both, _norm64(x_out, kind, weight, bias, 1e-6))
        bare = _norm(kind, d, affine=False)
        _check_int8((da.rmsnorm_int8 if kind == "rms" else da.layernorm_int8)(x, bare), _norm64(x, kind, None, None, 1e-6))


@pytest.mark.parametrize("d", [40, 512, 1500, 9000])
def test_int8_rows_do_not_depend_on_layout(d: int) -> None:
    """Batches, single rows, slices that start off a 16-byte boundary, strided and broadcast rows: the same bits."""
    norm = _norm("rms", d)
    x, branch = _randn(6, d, seed=1), _randn(6, d, seed=2, dtype=BF16)
    x_out, want = da.add_rmsnorm_int8(x, branch, norm)
    for make in (lambda t: F.pad(t, (1, 2))[:, 1:-2], lambda t: t.t().contiguous().t(), lambda t: F.pad(t, (0, 8))[:, :d]):
        o, got = da.add_rmsnorm_int8(make(x), make(branch), norm)
        assert torch.equal(o, x_out) and torch.equal(got.values, want.values)
        # the mean of squares is added in another order when elements are loaded one by one
        assert (got.scale - want.scale).abs().le(1e-6 * want.scale).all()
    o, got = da.add_rmsnorm_int8(x.view(2, 3, d), branch.view(2, 3, d), norm)
    assert got.values.shape == (2, 3, d) and got.scale.shape == (2, 3) and o.shape == (2, 3, d)
    assert torch.equal(got.values.reshape(6, d), want.values) and torch.equal(got.scale.view(6), want.scale)
    one = da.quantize_int8(x[4])
    assert one.values.shape == (d,) and one.scale.shape == ()
    assert torch.equal(one.values, da.quantize_int8(x).values[4])
    same = da.quantize_int8(x[:1].expand(5, d))
    assert torch.equal(same.values, one_row := same.values[:1].expand(5, d)) and one_row.shape == (5, d)


@pytest.mark.parametrize("d", [512, 1501, 8190])
def test_int8_rows_round_as_separate_operations_do(d: int) -> None:
    """q = rint(v * (127 / max|v|)) with each operation rounded to fp32, in every variant and bit for bit."""
    x = _randn(4000, d, seed=d)
    norm = _norm("rms", d)
    for rows, v in ((da.quantize_int8(x), x), (da.rmsnorm_int8(x, norm), x * norm.weight),
                    (da.quantize_int8(F.pad(x, (1, 0))[:, 1:]), x)):
        amax = v.abs().amax(1, keepdim=True)
        q = torch.round(v * (torch.full_like(amax, 127.0) / amax))
        assert torch.equal(rows.values.float(), q)


def test_int8_rows_of_zeros_tiny_and_non_finite_rows() -> None:
    d = 520
    x = _randn(9, d, seed=5)
    x[1] = 0
    x[2] = 1e-38
    x[3, 17] = float("nan")
    x[4, 519] = float("inf")
    x[5, 0] = -float("inf")
    x[6] = 0
    x[6, 400] = 1e-30
    for rows in (da.quantize_int8(x), da.rmsnorm_int8(x, _norm("rms", d)), da.layernorm_int8(x, _norm("layer", d)),
                 da.quantize_int8(F.pad(x, (1, 0))[:, 1:])):
        got = rows.dequantize()
        for r in (3, 4, 5):
            assert got[r].isnan().all() and not rows.scale[r].isfinite(), r
        for r in (0, 1, 2, 6, 7, 8):
            assert got[r].isfinite().all(), r
    rows = da.quantize_int8(x)
    assert rows.scale[1] == 0 and rows.values[1].eq(0).all()
    assert rows.values[6, 400] == 127 and rows.values[6].count_nonzero() == 1
    assert rows.scale[2] == 0  # 127 / 1e-38 is no fp32 number
    # eps = 0 on a row of zeros: 1 / sqrt(0) never reaches the values
    rows = da.rmsnorm_int8(torch.zeros(2, d, device="cuda"), nn.RMSNorm(d, eps=0.0).cuda().requires_grad_(False))
    assert rows.scale.eq(0).all() and rows.values.eq(0).all()


def test_int8_rows_empty_and_dequantize() -> None:
    rows = da.quantize_int8(torch.empty(0, 48, device="cuda"))
    assert rows.values.shape == (0, 48) and rows.scale.shape == (0,) and rows.dequantize().shape == (0, 48)
    for d in (1, 7, 64, 1001):
        rows = da.quantize_int8(_randn(11, d, seed=d))
        for dtype in (F32, BF16, F16):
            want = (rows.values.float() * rows.scale[:, None]).to(dtype)
            assert torch.equal(rows.dequantize(dtype), want)


def test_int8_rows_refusals() -> None:
    x, norm = _randn(4, 32), _norm("rms", 32)
    with pytest.raises(ValueError):
        da.rmsnorm_int8(x.cpu(), norm)
    with pytest.raises(ValueError):
        da.rmsnorm_int8(x.double(), norm)
    with pytest.raises(ValueError):
        da.rmsnorm_int8(x, _norm("rms", 33))
    with pytest.raises(ValueError):
        da.rmsnorm_int8(x, _norm("layer", 32))
    with pytest.raises(ValueError):
        da.layernorm_int8(x, norm)
    with pytest.raises(ValueError):
        da.add_rmsnorm_int8(x, x[:2], norm)
    with pytest.raises(ValueError):
        da.quantize_int8(torch.empty(4, 0, device="cuda"))
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        da.quantize_int8(x.clone().requires_grad_())


# ----------------------------------------------------------------------------- int8 product
def _gelu64(z: torch.Tensor) -> torch.Tensor:
    return z * torch.special.ndtr(z)


def _check_linear(x: da.Int8Rows, w: da.Int8Rows, bias, gelu: bool, dtype) -> None:
    y = da.int8_linear(x, w, bias, gelu=gelu, dtype=dtype)
    acc = x.values.double() @ w.values.double().t()
    z = acc * x.scale.double()[..., None] * w.scale.double()
    size = z.abs()
    if bias is not None:
        z = z + bias.double()
        size = size + bias.double().abs()
    want = _gelu64(z) if gelu else z
    allowed = 4 * 2.0**-24 * size * (1.2 if gelu else 1.0) + ROUNDING[dtype] * want.abs() * 1.01 + SMALLEST[dtype]
    if gelu:
        allowed = allowed + CDF * z.abs()
    assert y.dtype == dtype and y.shape == want.shape
    assert (y.double() - want).abs().le(allowed).all()


LINEAR_SHAPES = [(1, 1, 1), (1, 512, 1536), (1, 1536, 512), (2, 33, 5), (7, 100, 130), (16, 256, 256), (24, 4096, 512),
                 (31, 1000, 765), (64, 512, 1000), (65, 130, 128), (5, 1100, 200), (40, 2250, 129), (100, 48, 300), (129, 2048, 257), (256, 512, 1536),
                 (300, 96, 1), (511, 1024, 520), (1000, 520, 1032), (2100, 512, 1536), (4097, 64, 768)]


@pytest.mark.parametrize(("rows", "k", "n"), LINEAR_SHAPES)
def test_int8_linear_matches_its_definition(rows: int, k: int, n: int) -> None:
    w = da.quantize_int8(_randn(n, k, seed=1) * k**-0.5)
    x = da.quantize_int8(_randn(rows, k, seed=2, dtype=BF16))
    bias = _randn(n, seed=3)
    for gelu in (False, True):
        for dtype in (F32, BF16, F16):
            _check_linear(x, w, bias if dtype != F16 else None, gelu, dtype)
    _check_linear(x, w, bias.to(BF16), False, BF16)


@pytest.mark.parametrize(("rows", "k", "n"), [(20_011, 80, 1029), (15_000, 1030, 1288), (9_001, 1600, 1501)])
def test_int8_linear_of_many_tiles(rows: int, k: int, n: int) -> None:
    """Several output tiles for each pair of SMs, ragged at both edges, with scales and biases at odd addresses."""
    w = da.quantize_int8(_randn(n, k, seed=1) * k**-0.5)
    x = da.quantize_int8(_randn(rows, k, seed=2, dtype=BF16))
    bias = _randn(n + 1, seed=3)
    w_odd = da.Int8Rows(w.values, torch.cat((w.scale[:1], w.scale))[1:])
    for gelu in (False, True):
        _check_linear(x, w, bias[:-1], gelu, BF16)
        _check_linear(x, w, None, gelu, F16)
        _check_linear(x, w_odd, bias[1:], gelu, F32)
        _check_linear(x, w_odd, bias[1:].to(F16), gelu, BF16)
    alone = da.Int8Rows(x.values[-300:-44].contiguous(), x.scale[-300:-44].contiguous())
    assert torch.equal(da.int8_linear(x, w, bias[:-1], gelu=True)[-300:-44], da.int8_linear(alone, w, bias[:-1], gelu=True))


@pytest.mark.parametrize(("rows", "n"), [(2, 3), (40, 130), (300, 520)])
def test_int8_linear_sums_exactly_at_the_largest_inner_size(rows: int, n: int) -> None:
    k = eight_bit.MAX_INNER
    x = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[:, 5] = 127
    w[-1] = 127
    one = torch.ones(rows, device="cuda")
    y = da.int8_linear(da.Int8Rows(x, one), da.Int8Rows(w, torch.ones(n, device="cuda")), dtype=F32)
    want = torch.full((n,), 128 * 128 * (k - 1) - 128 * 127, dtype=torch.float64)
    want[-1] = -128 * 127 * k
    assert torch.equal(y, want.float().cuda().expand(rows, n))


def test_int8_linear_layouts_and_batches() -> None:
    k, n = 200, 96
    x = torch.randint(-127, 128, (5, 6, k), dtype=torch.int8, device="cuda", generator=_gen(1))
    xs = torch.rand(5, 6, device="cuda", generator=_gen(2)) + 0.1
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=_gen(3))
    ws = torch.rand(n, device="cuda", generator=_gen(4)) + 0.1
    want = da.int8_linear(da.Int8Rows(x, xs), da.Int8Rows(w, ws), dtype=F32)
    assert want.shape == (5, 6, n)
    flat = da.int8_linear(da.Int8Rows(x.view(30, k), xs.view(30)), da.Int8Rows(w, ws), dtype=F32)
    assert torch.equal(flat.view(5, 6, n), want)
    shifted = F.pad(x.float(), (3, 1)).to(torch.int8)[..., 3:-1]            # rows off 16-byte boundaries
    turned = w.t().contiguous().t()                                        # a column-major weight
    spread = torch.stack((xs, xs), -1)[..., 0]                              # strided scales
    assert torch.equal(da.int8_linear(da.Int8Rows(shifted, spread), da.Int8Rows(turned, ws), dtype=F32), want)
    one = da.int8_linear(da.Int8Rows(x[2, 3], xs[2, 3]), da.Int8Rows(w, ws), dtype=F32)
    assert one.shape == (n,) and torch.equal(one, want[2, 3])
    same = da.int8_linear(da.Int8Rows(x[:1, :1].expand(1, 4, k), xs[:1, :1].expand(1, 4)), da.Int8Rows(w, ws), dtype=F32)
    assert torch.equal(same, want[:1, :1].expand(1, 4, n))
    assert da.int8_linear(da.Int8Rows(x[:0], xs[:0]), da.Int8Rows(w, ws)).shape == (0, 6, n)


@pytest.mark.parametrize("rows", [1, 20, 700])
def test_int8_linear_row_by_row_equals_the_batch_and_a_bad_row_stays_alone(rows: int) -> None:
    """The product is exact, so a row's result does not depend on the rows beside it or on how many there are."""
    k, n = 384, 300
    w = da.quantize_int8(_randn(n, k, seed=1))
    x = _randn(rows, k, seed=2)
    x[rows // 2, 7] = float("nan")
    xq = da.quantize_int8(x)
    y = da.int8_linear(xq, w, gelu=True)
    assert y[rows // 2].isnan().all()
    for r in {0, rows // 3, rows - 1} - {rows // 2}:
        alone = da.int8_linear(da.Int8Rows(xq.values[r:r + 1], xq.scale[r:r + 1]), w, gelu=True)
        assert torch.equal(alone[0], y[r]) and y[r].isfinite().all()


def test_int8_linear_on_another_stream() -> None:
    w = da.quantize_int8(_randn(640, 512, seed=1))
    x = _randn(300, 512, seed=2)
    want = da.int8_linear(da.quantize_int8(x), w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            got = da.int8_linear(da.quantize_int8(x), w)
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        assert ops.device_status() == 0


def test_int8_linear_refusals() -> None:
    w, x = da.quantize_int8(_randn(64, 32)), da.quantize_int8(_randn(4, 32))
    bad = [(da.Int8Rows(x.values.to(torch.int32), x.scale), w, None), (da.Int8Rows(x.values, x.scale.half()), w, None),
           (da.Int8Rows(x.values, x.scale[:2]), w, None), (x, da.quantize_int8(_randn(64, 31)), None),
           (x, da.Int8Rows(w.values[None], w.scale[None]), None), (x, w, _randn(63)), (x, w, _randn(64).double()),
           (da.Int8Rows(x.values.cpu(), x.scale.cpu()), w, None)]
    for a, b, bias in bad:
        with pytest.raises(ValueError):
            da.int8_linear(a, b, bias)
    with pytest.raises(ValueError):
        da.int8_linear(x, w, dtype=torch.float64)
    long = torch.zeros(1, eight_bit.MAX_INNER + 1, dtype=torch.int8, device="cuda")
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        da.int8_linear(da.Int8Rows(long, one), da.Int8Rows(long, one))
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        da.int8_linear(x, w, _randn(64).requires_grad_())


# ----------------------------------------------------------------------------- checkpoints
def _kept64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Values [rows, blocks * 32] and exponents [rows, blocks] by the definition."""
    low, high = (-24, 9) if x.dtype == F16 else (-126, 121)
    d = x.shape[-1]
    v = F.pad(x.double().reshape(-1, d), (0, -d % 32)).unflatten(1, (-1, 32))
    a = v.abs().amax(2, keepdim=True)
    e = torch.full_like(a, low)
    for candidate in range(high, low - 1, -1):
        e = torch.where(a <= 127 * 2.0**candidate, torch.full_like(e, candidate), e)
    e = torch.where(a > 127 * 2.0**high, torch.full_like(e, high), e)
    q = (v / torch.exp2(e)).round().clamp(-127, 127)
    bad = ~a.isfinite()
    q, e = torch.where(bad, torch.zeros_like(q), q), torch.where(bad, torch.full_like(e, -128), e)
    return q.flatten(1).to(torch.int8), e[..., 0].to(torch.int8)


def _activation(rows: int, d: int, dtype, seed: int) -> torch.Tensor:
    """Normal values whose blocks lie between the dtype's smallest and largest numbers, some of them bad."""
    x = _randn(rows, d, seed=seed)
    g = _gen(seed + 1)
    top = 15 if dtype == F16 else 126
    size = torch.randint(-top - 12, top, (rows, -(-d // 32)), device="cuda", generator=g).double()
    size = torch.where(torch.rand(size.shape, device="cuda", generator=g) < 0.6, torch.zeros_like(size), size)
    big = torch.finfo(dtype).max
    x = (x.double() * torch.exp2(size).repeat_interleave(32, 1)[:, :d]).clamp(-big, big).to(dtype)
    flat = x.view(-1)
    flat[::997] = 0
    if flat.numel() > 3000:
        flat[1234], flat[2345], flat[777] = float("nan"), float("inf"), -float("inf")
        flat[1000], flat[1001] = big, -big
    return x


CHECKPOINT_SHAPES = [(1, 1), (1, 512), (3, 31), (5, 33), (40, 64), (33, 100), (129, 1536), (70, 1000), (2, 5000)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "d"), CHECKPOINT_SHAPES)
def test_checkpoint_is_exact(rows: int, d: int, dtype) -> None:
    x = _activation(rows, d, dtype, seed=rows + d)
    kept = da.checkpoint8(x)
    q, e = _kept64(x)
    assert torch.equal(kept.exponent, e) and torch.equal(kept.values, q)
    assert kept.shape == (rows, d) and kept.dtype == dtype
    stands = q.double() * torch.where(e == -128, torch.full_like(e.double(), math.nan), torch.exp2(e.double())) \
        .repeat_interleave(32, 1)
    got = kept.restore()
    assert got.dtype == dtype and torch.equal(got.double().nan_to_num(nan=1e300), stands[:, :d].nan_to_num(nan=1e300))
    for moved in (F.pad(x, (1, 1))[:, 1:-1], x.t().contiguous().t()):
        again = da.checkpoint8(moved)
        assert torch.equal(again.values, q) and torch.equal(again.exponent, e)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "d"), CHECKPOINT_SHAPES)
def test_gelu_checkpoint_forward(rows: int, d: int, dtype) -> None:
    z = (2.5 * _randn(rows, d, seed=d)).to(dtype)
    h, kept = da.gelu_checkpoint8(z)
    q, e = _kept64(z)
    assert torch.equal(kept.values, q) and torch.equal(kept.exponent, e)
    want = _gelu64(z.double())
    assert (h.double() - want).abs().le(1.01 * ROUNDING[dtype] * want.abs() + CDF * z.double().abs() + SMALLEST[dtype]).all()
    moved, _ = da.gelu_checkpoint8(F.pad(z, (1, 1))[:, 1:-1])
    assert torch.equal(moved, h)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "d"), CHECKPOINT_SHAPES)
def test_gelu_checkpoint_backward(rows: int, d: int, dtype) -> None:
    z = (2.5 * _randn(rows, d, seed=d)).to(dtype)
    dh = _randn(rows, d, seed=d + 1, dtype=dtype)
    kept = da.checkpoint8(z)
    dz, h = da.gelu_checkpoint8_backward(dh, kept)
    zk = kept.restore().double()
    slope = torch.special.ndtr(zk) + zk * torch.exp(-zk * zk / 2) / math.sqrt(2 * math.pi)
    want = dh.double() * slope
    allowed = 1.01 * ROUNDING[dtype] * want.abs() + 2 * CDF * (1 + zk.abs()) * dh.double().abs() + SMALLEST[dtype]
    assert (dz.double() - want).abs().le(allowed).all()
    want = _gelu64(zk)
    assert (h.double() - want).abs().le(1.01 * ROUNDING[dtype] * want.abs() + CDF * zk.abs() + SMALLEST[dtype]).all()
    # the slope against differences of GELU itself
    step = 1e-4
    slope = (_gelu64(zk + step) - _gelu64(zk - step)) / (2 * step)
    ones, _ = da.gelu_checkpoint8_backward(torch.ones_like(dh), kept)
    assert (ones.double() - slope).abs().le(1.01 * ROUNDING[dtype] * slope.abs() + 2 * CDF * (1 + zk.abs()) + 1e-7).all()
    # another layout of dh, the same bits
    moved, _ = da.gelu_checkpoint8_backward(dh.t().contiguous().t(), kept)
    assert torch.equal(moved, dz)


WGRAD_SHAPES = [(1, 1, 1), (3, 8, 40), (64, 128, 128), (100, 33, 65), (130, 392, 1000), (257, 256, 512), (1000, 1536, 128),
                (1025, 7, 520), (4096, 512, 256), (5001, 136, 200), (20000, 128, 384)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "n", "k"), WGRAD_SHAPES)
def test_weight_grad_from_a_checkpoint(rows: int, n: int, k: int, dtype) -> None:
    x, dy = _randn(rows, k, seed=1, dtype=dtype), _randn(rows, n, seed=2, dtype=dtype)
    kept = da.checkpoint8(x)
    xk = kept.restore().double()
    want = dy.double().t() @ xk
    size = dy.double().abs().t() @ xk.abs()
    # every addition of 16 products into the sum, and every partial sum, may round (or cut) at 2^-23
    allowed = 2.0**-23 * (rows / 16 + 64) * size
    for out in (F32, dtype):
        dw = da.weight_grad_checkpoint8(dy, kept, out)
        assert dw.dtype == out and dw.shape == (n, k)
        assert (dw.double() - want).abs().le(allowed + 1.01 * ROUNDING[out] * want.abs() + SMALLEST[out]).all()
        assert torch.equal(dw, da.weight_grad_checkpoint8(dy, kept, out)), "two runs differ"
    moved = F.pad(dy, (1, 2))[:, 1:-2]
    assert torch.equal(da.weight_grad_checkpoint8(moved, kept, F32), da.weight_grad_checkpoint8(dy, kept, F32))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("rows", "n", "k"), [(1, 9, 40), (2, 1, 33), (77, 129, 64), (700, 1001, 130), (6000, 777, 520)])
def test_weight_grad_of_odd_widths_in_any_layout(rows: int, n: int, k: int, dtype) -> None:
    """dY off 16-byte rows, at any address: the bits of the same dY laid out on them."""
    dy, kept = _randn(rows, n, seed=2, dtype=dtype), da.checkpoint8(_randn(rows, k, seed=1, dtype=dtype))
    want = da.weight_grad_checkpoint8(F.pad(dy, (0, -n % 8))[:, :n], kept, F32)
    xk = kept.restore().double()
    allowed = 2.0**-23 * (rows / 16 + 64) * (dy.double().abs().t() @ xk.abs()) + 2.0**-150
    assert (want.double() - dy.double().t() @ xk).abs().le(1.01 * 2.0**-24 * want.double().abs() + allowed).all()
    flat = torch.full((rows * (n + 5) + 16,), math.nan, dtype=dtype, device="cuda")
    for off, ld in ((0, n), (1, n), (7, n), (3, n + 5), (0, n + 3)):
        moved = flat[off:].as_strided((rows, n), (ld, 1))
        flat.fill_(math.nan)
        moved.copy_(dy)
        assert torch.equal(da.weight_grad_checkpoint8(moved, kept, F32), want)
    one = dy[:1].expand(rows, n)
    assert torch.equal(da.weight_grad_checkpoint8(one, kept, F32), da.weight_grad_checkpoint8(one.contiguous(), kept, F32))


def test_weight_grad_of_no_rows_and_of_bad_blocks() -> None:
    kept = da.checkpoint8(torch.empty(0, 64, dtype=BF16, device="cuda"))
    dw = da.weight_grad_checkpoint8(torch.empty(0, 16, dtype=BF16, device="cuda"), kept)
    assert dw.shape == (16, 64) and dw.eq(0).all()
    x = _randn(200, 96, seed=1, dtype=BF16)
    x[77, 40] = float("inf")
    dw = da.weight_grad_checkpoint8(_randn(200, 16, seed=2, dtype=BF16), da.checkpoint8(x), F32)
    assert dw[:, 32:64].isnan().all() and dw[:, :32].isfinite().all() and dw[:, 64:].isfinite().all()


def test_checkpoint_extremes_in_products() -> None:
    """Blocks at the ends of the exponent range multiply as the values they stand for."""
    for dtype, low, high in ((F16, 2.0**-24, 2.0**9), (BF16, 2.0**-120, 2.0**100)):
        x = torch.zeros(48, 64, dtype=dtype, device="cuda")
        x[:, :32] = low * 3
        x[:, 32:] = high * 100
        kept = da.checkpoint8(x)
        assert torch.equal(kept.restore(), x)
        dy = torch.ones(48, 8, dtype=dtype, device="cuda")
        dw = da.weight_grad_checkpoint8(dy, kept, F32)
        assert torch.equal(dw[:, :32], torch.full_like(dw[:, :32], 48 * low * 3))
        assert torch.equal(dw[:, 32:], torch.full_like(dw[:, 32:], 48 * high * 100))


def test_checkpoint_refusals() -> None:
    x = _randn(8, 64, dtype=BF16)
    kept = da.checkpoint8(x)
    with pytest.raises(ValueError):
        da.checkpoint8(x.float())
    with pytest.raises(ValueError):
        da.checkpoint8(x.cpu())
    with pytest.raises(ValueError):
        da.gelu_checkpoint8_backward(x[:4], kept)
    with pytest.raises(ValueError):
        da.gelu_checkpoint8_backward(x.half(), kept)
    with pytest.raises(ValueError):
        da.weight_grad_checkpoint8(x.half(), kept)
    with pytest.raises(ValueError):
        da.weight_grad_checkpoint8(x[:4], kept)
    with pytest.raises(ValueError):
        da.weight_grad_checkpoint8(x, kept, F16)
    with pytest.raises(ValueError):
        da.Checkpoint8(kept.values[:, :32], kept.exponent, (8, 64), BF16).restore()
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        da.gelu_checkpoint8(x.clone().requires_grad_())
    with pytest.raises(NotImplementedError):
        da.linear_checkpoint8(x, nn.Linear(64, 128).cuda().to(BF16))


# ----------------------------------------------------------------------------- training through checkpoints
def _cos(a: torch.Tensor, b: torch.Tensor) -> float:
    return F.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_checkpoint8_gradients(dtype) -> None:
    torch.manual_seed(1)
    layer = nn.Linear(256, 384).cuda()
    x = _randn(3, 70, 256, seed=1)
    dy = _randn(3, 70, 384, seed=2)
    with torch.enable_grad(), torch.autocast("cuda", dtype=dtype):
        xr = x.clone().requires_grad_()
        y = da.linear_checkpoint8(xr, layer)
        plain = ops.linear(x, layer)
    assert torch.equal(y, plain)
    y.backward(dy.to(dtype))
    xh = da.checkpoint8(x.to(dtype)).restore().double().reshape(-1, 256)
    g = dy.to(dtype).double().reshape(-1, 384)
    want = g.t() @ xh
    assert (layer.weight.grad.double() - want).abs().le(2.0**-23 * 80 * (g.abs().t() @ xh.abs())).all()
    assert _cos(xr.grad, g @ layer.weight.to(dtype).double()) > 0.99999
    assert (layer.bias.grad.double() - g.sum(0)).abs().le(2.0**-8 * g.abs().sum(0)).all()
    # against differences: the loss <y, dy> is linear in W, so its change along V is <dW, V> up to what the
    # checkpoint changed of x, at most half a unit 2^e of each value
    v = _randn(384, 256, seed=5).double()
    x64 = x.to(dtype).double().reshape(-1, 256)
    change = ((x64 @ v.t()) * g).sum()
    half_unit = torch.exp2(da.checkpoint8(x.to(dtype)).exponent.double() - 1).repeat_interleave(32, 1)
    allowed = ((g.abs() @ v.abs()) * half_unit).sum()
    assert ((layer.weight.grad.double() * v).sum() - change).abs() <= allowed


def test_feedforward_checkpoint8_gradients_and_memory() -> None:
    torch.manual_seed(2)
    first, second = nn.Linear(256, 768).cuda(), nn.Linear(768, 256).cuda()
    x, dout = _randn(2, 300, 256, seed=1), _randn(2, 300, 256, seed=2)

    def grads(fn, saved: list):
        for p in (*first.parameters(), *second.parameters()):
            p.grad = None
        xr = x.clone().requires_grad_()
        with torch.enable_grad(), torch.autocast("cuda", dtype=BF16), torch.autograd.graph.saved_tensors_hooks(
                lambda t: saved.append(t.numel() * t.element_size()) or t, lambda t: t):
            y = fn(xr, first, second)
        y.backward(dout.to(BF16))
        return y, [xr.grad] + [p.grad.clone() for p in (*first.parameters(), *second.parameters())]

    kept, full = [], []
    y8, g8 = grads(da.feedforward_checkpoint8, kept)
    y16, g16 = grads(ops.feedforward, full)
    assert _cos(y8, y16) > 0.99999
    for a, b in zip(g8, g16):
        # the checkpoint rounds a block's values by at most 1/128 of its largest: about 1 % of a normal value
        assert _cos(a, b) > 0.9995
    weights = 2 * 2 * 256 * 768
    assert sum(kept) - weights < 0.33 * (sum(full) - weights)
    again = grads(da.feedforward_checkpoint8, [])[1]
    assert all(torch.equal(a, b) for a, b in zip(g8, again)), "two runs differ"


# ----------------------------------------------------------------------------- capture, the other device side, long tensors
def test_eight_bit_calls_replay_from_a_graph() -> None:
    x, branch = _randn(33, 512, seed=1), _randn(33, 512, seed=2, dtype=BF16)
    norm, w = _norm("rms", 512), da.quantize_int8(_randn(640, 512, seed=3))
    dy = _randn(33, 128, seed=4, dtype=BF16)

    def step():
        x_out, rows = da.add_rmsnorm_int8(x, branch, norm)
        h, kept = da.gelu_checkpoint8(da.int8_linear(rows, w))
        dz, _ = da.gelu_checkpoint8_backward(h, kept)
        return x_out, h, dz, da.weight_grad_checkpoint8(dy, kept)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (7, 8):
        x.copy_(_randn(33, 512, seed=seed))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_both_host_paths_give_the_same(monkeypatch) -> None:
    """The extension's calls against the Python ones, which take what it leaves."""
    class Nothing:
        def __getattr__(self, name):
            return lambda *args: None

    def results():
        x, branch = _randn(2, 9, 200, seed=1), _randn(2, 9, 200, seed=2, dtype=F16)
        x_out, rows = da.add_layernorm_int8(x, branch, _norm("layer", 200))
        bare = da.rmsnorm_int8(x, _norm("rms", 200, affine=False))
        y = da.int8_linear(rows, da.quantize_int8(_randn(40, 200, seed=3)), _randn(40, seed=4), gelu=True, dtype=F16)
        h, kept = da.gelu_checkpoint8(y)
        dz, again = da.gelu_checkpoint8_backward(h, kept)
        dw = da.weight_grad_checkpoint8(h, da.checkpoint8(x.half()), F32)
        return [x_out, *rows, *bare, rows.dequantize(BF16), y, h, kept.values, kept.exponent, dz, again, dw]

    fast = results()
    monkeypatch.setattr(eight_bit, "_host_module", Nothing())
    slow = results()
    assert all(a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(fast, slow))


def test_tensors_of_more_than_2_to_the_31_elements() -> None:
    """Offsets past 32 bits: the last rows of tensors of 2.5e9 elements against the same rows alone."""
    rows, d = 300_000, 8192
    x = torch.empty(rows, d, dtype=BF16, device="cuda")
    tail = _randn(500, d, seed=1, dtype=BF16)
    x.zero_()[-500:] = tail
    alone, got = da.quantize_int8(tail), da.quantize_int8(x)
    assert torch.equal(got.values[-500:], alone.values) and torch.equal(got.scale[-500:], alone.scale)
    assert torch.equal(got.dequantize(BF16)[-500:], alone.dequantize(BF16))
    w = da.quantize_int8(_randn(300, d, seed=2))
    assert torch.equal(da.int8_linear(got, w)[-500:], da.int8_linear(alone, w))
    del got
    h, kept = da.gelu_checkpoint8(x)
    h1, kept1 = da.gelu_checkpoint8(tail)
    assert torch.equal(h[-500:], h1) and torch.equal(kept.values[-500:], kept1.values)
    assert torch.equal(kept.restore()[-500:], kept1.restore())
    dz, _ = da.gelu_checkpoint8_backward(x, kept)
    assert torch.equal(dz[-500:], da.gelu_checkpoint8_backward(tail, kept1)[0])
    del h, dz
    few = _randn(rows, 8, seed=3, dtype=BF16)
    # x is zero in all other rows; the last 500 rows add in another order, in one split
    dw, dw1 = da.weight_grad_checkpoint8(few, kept, F32), da.weight_grad_checkpoint8(few[-500:], kept1, F32)
    size = few[-500:].float().abs().t() @ kept1.restore().float().abs()
    assert (dw - dw1).abs().le(2.0**-23 * 100 * size).all()
    back = da.weight_grad_checkpoint8(x, da.checkpoint8(few), F32)  # dy of 2.5e9 elements
    ones = da.weight_grad_checkpoint8(tail, da.checkpoint8(few[-500:]), F32)
    size = tail.float().abs().t() @ few[-500:].float().abs()
    assert (back - ones).abs().le(2.0**-23 * 100 * size).all()
    out = da.int8_linear(da.Int8Rows(torch.ones(rows, 16, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda")),
                         da.Int8Rows(torch.ones(d, 16, dtype=torch.int8, device="cuda"), torch.ones(d, device="cuda")))
    assert out[-500:].eq(16).all() and out[:, -1].eq(16).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 40, 1000, 1536])
def test_checkpoint_layouts_give_the_same_bits(d: int, dtype) -> None:
    """Rows on 16-byte words of a wider tensor, rows off them, and one row for all."""
    rows = 67
    z, dh = (2.5 * _randn(rows, d, seed=d)).to(dtype), _randn(rows, d, seed=d + 1, dtype=dtype)
    h, kept = da.gelu_checkpoint8(z)
    dz, again = da.gelu_checkpoint8_backward(dh, kept)
    for left, right in ((8, 16), (8, 1), (3, 5)):
        wide_z, wide_dh = (F.pad(t, (left, right))[:, left:-right] for t in (z, dh))
        h1, kept1 = da.gelu_checkpoint8(wide_z)
        assert torch.equal(h1, h) and torch.equal(kept1.values, kept.values) and torch.equal(kept1.exponent, kept.exponent)
        dz1, again1 = da.gelu_checkpoint8_backward(wide_dh, kept)
        assert torch.equal(dz1, dz) and torch.equal(again1, again)
    h1, kept1 = da.gelu_checkpoint8(z[:1].expand(rows, d))
    assert torch.equal(h1, h[:1].expand(rows, d)) and torch.equal(kept1.values, kept.values[:1].expand(rows, -1))


@pytest.mark.parametrize("d", [1, 31, 33, 1000, 1001, 1024])
def test_checkpoint_results_in_place_of_their_input(d: int) -> None:
    """The C entries, with an output at the address of the input; and values restored to fp32."""
    rows = 700
    z, dh = (2.5 * _randn(rows, d, seed=d)).to(BF16), _randn(rows, d, seed=d + 1, dtype=BF16)
    h, kept = da.gelu_checkpoint8(z)
    dz, again = da.gelu_checkpoint8_backward(dh, kept)
    q, e = torch.empty_like(kept.values), torch.empty_like(kept.exponent)
    own, code = z.clone(), eight_bit._CODES[BF16]
    eight_bit._launch(0, "da_checkpoint8", own.data_ptr(), code, d, rows, d, 1, own.data_ptr(), d, q.data_ptr(), e.data_ptr())
    assert torch.equal(own, h) and torch.equal(q, kept.values) and torch.equal(e, kept.exponent)
    kept_args = (q.data_ptr(), e.data_ptr(), rows, d)
    for dz_in_place in (True, False):
        own, other = dh.clone(), torch.empty_like(dh)
        a, b = (own, other) if dz_in_place else (other, own)
        eight_bit._launch(0, "da_checkpoint8_gelu_bwd", own.data_ptr(), code, d, *kept_args, a.data_ptr(), d, b.data_ptr(), d)
        assert torch.equal(a, dz) and torch.equal(b, again)
    for ld in (d, d + 3, (d + 7) // 8 * 8 + 8):
        wide = torch.full((rows, ld), -7.0, device="cuda")
        eight_bit._launch(0, "da_checkpoint8_restore", *kept_args, wide.data_ptr(), eight_bit._CODES[F32], ld)
        assert torch.equal(wide[:, :d], kept.restore().float()) and wide[:, d:].eq(-7).all()


@pytest.mark.parametrize("d", [1, 8])
def test_checkpoint_of_more_rows_than_one_launch_takes(d: int) -> None:
    """A checkpoint pads rows to 32 columns: past 2^31 groups of 8, with offsets into it past 2^34."""
    rows = 2**29 + 5000
    ends = (2.5 * _randn(10_000, d, seed=d)).to(BF16)
    z = torch.zeros(rows, d, dtype=BF16, device="cuda")
    z[:10_000], z[-10_000:] = ends, ends
    h, kept = da.gelu_checkpoint8(z)
    h1, kept1 = da.gelu_checkpoint8(ends)
    dz1, _ = da.gelu_checkpoint8_backward(ends, kept1)
    back, back1 = kept.restore(), kept1.restore()
    dz, _ = da.gelu_checkpoint8_backward(z, kept)
    for part in (slice(None, 10_000), slice(-10_000, None)):
        assert torch.equal(h[part], h1) and torch.equal(back[part], back1) and torch.equal(dz[part], dz1)
        assert torch.equal(kept.values[part], kept1.values) and torch.equal(kept.exponent[part], kept1.exponent)
