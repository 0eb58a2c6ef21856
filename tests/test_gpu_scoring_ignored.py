"""Scores' gradient in rows whose token is none: exact zeros, whatever the row holds, unless its entropy counts."""

from __future__ import annotations

import math

import pytest
import torch

import double_attention_b200 as da

pytestmark = pytest.mark.gpu


def _rows(width: int, dtype: torch.dtype, shift: int) -> torch.Tensor:
    """Six rows: ordinary, NaN, all minus infinity, one plus infinity, one NaN, ordinary; off 16 bytes by ``shift`` elements."""
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(6, width + shift, device="cuda", generator=g).to(dtype)[:, shift:]
    x[1], x[2] = math.nan, -math.inf
    x[3, 3], x[4, width - 1] = math.inf, math.nan
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("width", "shift"), [(7, 0), (100, 0), (1001, 1), (5000, 0), (5000, 3)])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_a_row_without_a_token_passes_no_gradient(width, shift, dtype, with_entropy) -> None:
    x = _rows(width, dtype, shift).requires_grad_()
    tokens = torch.tensor([-100, -100, -100, -100, -100, 2], device="cuda")
    made = da.token_log_probs(x, tokens)
    g = torch.ones(6, device="cuda")
    if with_entropy:  # (not of the rows without a token)
        h = torch.zeros(6, device="cuda")
        h[5] = 0.5
        d, = torch.autograd.grad((made.log_probs, made.entropy), x, (g, h))
    else:
        d, = torch.autograd.grad(made.log_probs, x, g)
    assert not d[:5].any() and not d[:5].isnan().any()
    row = x.detach()[5].double().requires_grad_()
    lp = torch.log_softmax(row, 0)
    (lp[2] + (0.5 if with_entropy else 0.0) * -(lp.exp() * lp).sum()).backward()
    bound = torch.finfo(dtype).eps / 2 * row.grad.abs() + 1e-5 * (row.grad.abs() + lp.exp()) + 1e-7
    assert ((d[5].double() - row.grad).abs() <= bound).all()


def test_a_row_whose_entropy_counts_still_says_that_it_is_none() -> None:
    x = _rows(64, torch.float32, 0).requires_grad_()
    made = da.token_log_probs(x, torch.full((6,), -100, device="cuda"))
    d, = torch.autograd.grad(made.entropy.sum(), x)
    assert d[1:5].isnan().all() and d[0].isfinite().all() and d[5].isfinite().all() and d[0].any()


def test_a_zero_gradient_of_a_row_with_a_token_stays_what_a_softmax_gives() -> None:
    x = _rows(64, torch.float32, 0).requires_grad_()
    made = da.token_log_probs(x, torch.zeros(6, dtype=torch.long, device="cuda"))
    d, = torch.autograd.grad(made.log_probs, x, torch.zeros(6, device="cuda"))
    assert d[1:5].isnan().all() and not d[0].any()
