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
