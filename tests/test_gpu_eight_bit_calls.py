"""What the eight-bit operators take from their callers' modules and tensors: the default eps of a norm, gradients and
tangents that they have to refuse, layers that are more than their class, empty inputs.

Tolerances, fixed from the formulas: an int8 row is within half a step of the exact value plus the fp32 error of its
factors (2e-3 steps); a 16-bit module's own result is rounded at most twice.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import double_attention_b200 as da
from double_attention_b200 import ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _randn(*shape: int, seed: int = 0, dtype=F32) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    torch.cuda.synchronize()
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rms_norm_without_an_eps_takes_the_modules_own(dtype) -> None:
    """nn.RMSNorm(d) has eps None; rows small enough that another eps than the module's shows."""
    norm = nn.RMSNorm(512).cuda().to(dtype).requires_grad_(False)
    rounding = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}[dtype]
    for size in (1.0, 1e-3):
        x, branch = _randn(40, 512, seed=1, dtype=dtype) * size, _randn(40, 512, seed=2, dtype=dtype) * size
        x_out, added = da.add_rmsnorm_int8(x, branch, norm)
        for rows, want in ((da.rmsnorm_int8(x, norm), norm(x)), (added, norm(x_out))):
            got, want = rows.dequantize().double(), want.double()
            step = want.abs().amax(-1, keepdim=True) / 127
            assert (got - want).abs().le(0.502 * step + 2.02 * rounding * (want.abs() + 127 * step)).all()
            r = (x if rows is not added else x_out).double()
            exact = r / torch.sqrt(r.square().mean(-1, keepdim=True) + 2.0**-23)
            assert (got - exact).abs().le(0.502 * exact.abs().amax(-1, keepdim=True) / 127).all()
