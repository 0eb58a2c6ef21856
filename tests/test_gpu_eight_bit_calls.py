"""What the eight-bit operators take from their callers' modules and tensors: the default eps of a norm, gradients and
tangents that they have to refuse, layers that are more than their class, empty inputs.

Tolerances, fixed from the formulas: an int8 row is within half a step of the exact value plus the fp32 error of its
factors (2e-3 steps); a 16-bit module's own result is rounded at most twice.
"""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
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


def _rows_and_weight() -> tuple[da.Int8Rows, da.Int8Rows]:
    return da.quantize_int8(_randn(4, 32, seed=1)), da.quantize_int8(_randn(64, 32, seed=2))


def test_a_scale_that_requires_a_gradient_is_refused() -> None:
    """The result would have no graph, and the scale would silently get no gradient."""
    x, w = _rows_and_weight()
    learned = lambda rows: da.Int8Rows(rows.values, rows.scale.clone().requires_grad_())
    want, decoded = da.int8_linear(x, w), x.dequantize()
    for call in (lambda: da.int8_linear(learned(x), w), lambda: da.int8_linear(x, learned(w)),
                 lambda: learned(x).dequantize(), lambda: learned(x).dequantize(BF16)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        assert torch.equal(da.int8_linear(learned(x), learned(w)), want)
        assert torch.equal(learned(x).dequantize(), decoded)


def test_forward_mode_tangents_are_refused() -> None:
    x32, x16 = _randn(4, 32, seed=1), _randn(4, 32, seed=1, dtype=BF16)
    rms, layer = nn.RMSNorm(32).cuda().requires_grad_(False), nn.LayerNorm(32).cuda().requires_grad_(False)
    x, w = _rows_and_weight()
    kept, bias = da.checkpoint8(x16), _randn(64, seed=3)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: da.quantize_int8(dual(x32)), lambda: da.rmsnorm_int8(dual(x16), rms),
                     lambda: da.add_layernorm_int8(x32, dual(x32), layer), lambda: da.add_rmsnorm_int8(dual(x32), x32, rms),
                     lambda: da.int8_linear(da.Int8Rows(x.values, dual(x.scale)), w),
                     lambda: da.int8_linear(x, da.Int8Rows(w.values, dual(w.scale))),
                     lambda: da.int8_linear(x, w, dual(bias)), lambda: da.Int8Rows(x.values, dual(x.scale)).dequantize(),
                     lambda: da.checkpoint8(dual(x16)), lambda: da.gelu_checkpoint8(dual(x16)),
                     lambda: da.gelu_checkpoint8_backward(dual(x16), kept),
                     lambda: da.weight_grad_checkpoint8(dual(x16), kept)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
        # primal tensors, and duals where the mode is off, pass
        assert torch.equal(da.quantize_int8(x32).values, x.values)
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(da.quantize_int8(dual(x32)).values, x.values)


@pytest.mark.parametrize("loss", [lambda y: y.float().sum(), lambda y: y.float().square().sum()])
@pytest.mark.parametrize("kind", ["linear", "feedforward"])
def test_gradients_of_checkpointed_layers_raise_when_differentiated(kind: str, loss) -> None:
    """create_graph=True gives the first derivatives; a penalty on them must not pass as a constant."""
    torch.manual_seed(1)
    first, second = nn.Linear(256, 384).cuda().to(BF16), nn.Linear(384, 256).cuda().to(BF16)
    x = _randn(16, 256, seed=1, dtype=BF16).requires_grad_()
    params = list(first.parameters()) + (list(second.parameters()) if kind == "feedforward" else [])

    def forward():
        return loss(da.linear_checkpoint8(x, first) if kind == "linear" else da.feedforward_checkpoint8(x, first, second))

    plain = torch.autograd.grad(forward(), (x, *params))
    grads = torch.autograd.grad(forward(), (x, *params), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    for g in grads:
        assert g.requires_grad and not plain[0].requires_grad
        with pytest.raises(RuntimeError, match="no second derivative"):
            g.float().square().sum().backward(retain_graph=True)


def test_feedforward_keeps_its_input_for_the_first_weights_gradient_alone() -> None:
    torch.manual_seed(1)
    first, second = nn.Linear(256, 384).cuda().to(BF16), nn.Linear(384, 256).cuda().to(BF16)
    x, dout = _randn(100, 256, seed=1, dtype=BF16).requires_grad_(), _randn(100, 256, seed=2, dtype=BF16)

    def step() -> tuple[int, list]:
        kept: list = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
            y = da.feedforward_checkpoint8(x, first, second)
        wanted = [x, first.bias, *second.parameters()]
        return sum(kept), torch.autograd.grad(y, wanted, dout)

    full, grads = step()
    first.weight.requires_grad_(False)
    less, same = step()
    assert full - less == 100 * 256 * 33 // 32
    assert all(torch.equal(a, b) for a, b in zip(grads, same))


def test_weight_grad_with_a_checkpoint_without_dimensions_is_refused() -> None:
    x = torch.zeros(1, 32, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="takes a checkpoint"):
        da.weight_grad_checkpoint8(torch.zeros(8, dtype=BF16, device="cuda"), da.Checkpoint8(x, x[:, :1], (), BF16))
