"""The C entries of the eight-bit operators write their outputs' elements and nothing else: rows wider apart than they are
long, and buffers with more before and behind, keep what lies between and around.  The outputs equal those of the
dense call bit for bit."""

from __future__ import annotations

import pytest
import torch

import double_attention_b200 as da
from double_attention_b200 import eight_bit, ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODES = eight_bit._CODES
AROUND = 256  # elements before and behind


def _randn(*shape: int, seed: int = 0, dtype=F32) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    torch.cuda.synchronize()
    assert ops.device_status() == 0


class _Guarded:
    """Rows [rows, d] at stride ld inside a buffer of known bytes."""

    def __init__(self, rows: int, d: int, ld: int, dtype) -> None:
        self.buffer = torch.empty(2 * AROUND + (rows - 1) * ld + d, dtype=dtype, device="cuda")
        self.buffer.view(torch.int8).random_(-100, 100, generator=torch.Generator(device="cuda").manual_seed(rows))
        self.before = self.buffer.clone()
        self.at = lambda buffer: buffer.as_strided((rows, d), (ld, 1), AROUND)

    @property
    def rows(self) -> torch.Tensor:
        return self.at(self.buffer)

    def check(self) -> None:
        for buffer in (now := self.buffer.clone(), was := self.before.clone()):
            self.at(buffer).zero_()
        assert torch.equal(now.view(torch.int8), was.view(torch.int8)), "wrote outside its rows"


# few tokens; CTA pairs, with long K and with short; widths that end inside a 16-byte word, at it, and inside the first
@pytest.mark.parametrize(("m", "k"), [(5, 64), (700, 48), (3000, 200), (2500, 1600)])
@pytest.mark.parametrize("n", [2, 1283, 2047, 2304])
def test_products_leave_what_lies_between_rows(m: int, k: int, n: int) -> None:
    x, w = da.quantize_int8(_randn(m, k, seed=1)), da.quantize_int8(_randn(n, k, seed=2))
    bias = _randn(n, seed=3)
    for dtype in (F32, BF16, F16):
        for gelu in (False, True):
            want = da.int8_linear(x, w, bias, gelu=gelu, dtype=dtype)
            for ld in (n, n + 1, -(-n // 8) * 8, -(-n // 8) * 8 + 8):
                out = _Guarded(m, n, ld, dtype)
                eight_bit._launch(0, "da_gemm_i8", x.values.data_ptr(), x.values.stride(0), x.scale.data_ptr(),
                                  w.values.data_ptr(), w.values.stride(0), w.scale.data_ptr(), bias.data_ptr(), CODES[F32],
                                  int(gelu), out.rows.data_ptr(), ld, CODES[dtype], m, n, k,
                                  ops.workspace(x.scale.device).status.data_ptr())
                out.check()
                assert torch.equal(out.rows, want)


# widths of a warp's row and of a block's, on 16-byte rows and off them, and a row wider than registers hold
WIDTHS = [1, 7, 40, 501, 512, 1999, 4096, 16_400]


@pytest.mark.parametrize("d", WIDTHS)
def test_norms_leave_what_lies_between_rows(d: int) -> None:
    rows, eps, pitch = 37, 1e-6, -(-d // 16) * 16
    norm = torch.nn.RMSNorm(d, eps=eps).cuda().requires_grad_(False)
    for dtype, branch_dtype in ((F32, BF16), (BF16, BF16), (F16, F32)):
        x, branch = _randn(rows, d, seed=1, dtype=dtype), _randn(rows, d, seed=2, dtype=branch_dtype)
        x_out, want = da.add_rmsnorm_int8(x, branch, norm)
        for ld in (d, d + 1, pitch + 16):
            # (up to 7 bytes behind a row of q may be written where its stride has room for them)
            for ldq in (d, pitch, pitch + 16):
                out, scale = _Guarded(rows, d, ld, dtype), _Guarded(1, rows, rows, F32)
                q = _Guarded(rows, min(ldq, -(-d // 8) * 8), ldq, torch.int8)
                eight_bit._launch(0, "da_norm_int8", x.data_ptr(), CODES[dtype], d, branch.data_ptr(), CODES[branch_dtype], d,
                                  norm.weight.data_ptr(), CODES[F32], None, 0, eight_bit._RMS, rows, d, eps,
                                  out.rows.data_ptr(), ld, q.rows.data_ptr(), ldq, scale.rows.data_ptr())
                for guarded in (out, scale, q):
                    guarded.check()
                assert torch.equal(out.rows, x_out) and torch.equal(q.rows[:, :d], want.values)
                # (elements that are loaded one by one add their squares in another order)
                assert (scale.rows[0] - want.scale).abs().le(1e-6 * want.scale).all()
        decoded = want.dequantize(dtype)
        for ld in (d, d + 1, pitch + 16):
            out = _Guarded(rows, d, ld, dtype)
            eight_bit._launch(0, "da_dequant_int8", want.values.data_ptr(), pitch, want.scale.data_ptr(), rows, d,
                              out.rows.data_ptr(), CODES[dtype], ld)
            out.check()
            assert torch.equal(out.rows, decoded)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_checkpoints_leave_what_lies_between_rows(d: int, dtype) -> None:
    rows, blocks = 67, -(-d // 32)
    z, dh = _randn(rows, d, seed=1, dtype=dtype), _randn(rows, d, seed=2, dtype=dtype)
    h, kept = da.gelu_checkpoint8(z)
    dz, again = da.gelu_checkpoint8_backward(dh, kept)
    restored = kept.restore()
    for ld in (d, d + 1, -(-d // 8) * 8 + 8):
        out, q, e = _Guarded(rows, d, ld, dtype), _Guarded(1, rows * blocks * 32, 1, torch.int8), _Guarded(1, rows * blocks, 1, torch.int8)
        eight_bit._launch(0, "da_checkpoint8", z.data_ptr(), CODES[dtype], d, rows, d, 1, out.rows.data_ptr(), ld,
                          q.rows.data_ptr(), e.rows.data_ptr())
        back, slope, value = (_Guarded(rows, d, ld, dtype) for _ in range(3))
        eight_bit._launch(0, "da_checkpoint8_restore", q.rows.data_ptr(), e.rows.data_ptr(), rows, d, back.rows.data_ptr(),
                          CODES[dtype], ld)
        eight_bit._launch(0, "da_checkpoint8_gelu_bwd", dh.data_ptr(), CODES[dtype], d, q.rows.data_ptr(), e.rows.data_ptr(),
                          rows, d, slope.rows.data_ptr(), ld, value.rows.data_ptr(), ld)
        for guarded in (out, q, e, back, slope, value):
            guarded.check()
        assert torch.equal(q.rows.view_as(kept.values), kept.values) and torch.equal(e.rows.view_as(kept.exponent), kept.exponent)
        for guarded, want in ((out, h), (back, restored), (slope, dz), (value, again)):
            assert torch.equal(guarded.rows, want)


@pytest.mark.parametrize(("rows", "n", "k"), [(70, 9, 33), (700, 392, 1000), (3000, 777, 130), (300, 2304, 2300)])
def test_weight_gradients_leave_what_lies_between_rows(rows: int, n: int, k: int) -> None:
    dy, kept = _randn(rows, n, seed=1, dtype=BF16), da.checkpoint8(_randn(rows, k, seed=2, dtype=BF16))
    elems = int(eight_bit._lib.lib().da_checkpoint8_wgrad_workspace_elems(rows, n, k))
    for dtype in (F32, BF16):
        want = da.weight_grad_checkpoint8(dy, kept, dtype)
        for ld in (k, k + 1, -(-k // 8) * 8 + 8):
            out, work = _Guarded(n, k, ld, dtype), _Guarded(1, max(elems, 1), 1, F32)
            eight_bit._launch(0, "da_checkpoint8_wgrad", dy.data_ptr(), CODES[BF16], n, kept.values.data_ptr(),
                              kept.exponent.data_ptr(), rows, n, k, out.rows.data_ptr(), CODES[dtype], ld,
                              work.rows.data_ptr(), elems, ops.workspace(dy.device).status.data_ptr())
            out.check()
            work.check()
            assert torch.equal(out.rows, want)
