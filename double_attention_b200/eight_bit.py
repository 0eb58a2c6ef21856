"""Eight-bit operators: an int8 serving path and 8-bit activation checkpoints for training.

Serving.  A norm leaves its rows in int8 with one scale per token (:func:`add_rmsnorm_int8`,
:func:`add_layernorm_int8` and their forms without a branch), activations that no norm precedes go
through :func:`quantize_int8` -- as do the weights, once, with one scale per output channel -- and
:func:`int8_linear` multiplies the two on the int8 tensor cores, from a single token to long batches.
These operators have no backward; called on tensors that require a gradient, or that carry a forward-mode
tangent, they raise.

Training.  :func:`gelu_checkpoint8` keeps GELU's input in 8 bits (blocks of 32 columns sharing a
power-of-two scale) in place of the 16-bit tensor, :func:`gelu_checkpoint8_backward` and
:func:`weight_grad_checkpoint8` work from such a checkpoint, and :func:`linear_checkpoint8` and
:func:`feedforward_checkpoint8` put them together behind autograd: a Linear and the block's
feed-forward branch whose saved activations take 8 bits an element.

Every numeric step runs in the kernels of ``libda_b200.so``; unsupported inputs raise.
"""

from __future__ import annotations

import math
import warnings
from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib, ops
from ._lib import ptr

BLOCK = 32          # columns of a checkpoint that share one exponent
MAX_INNER = 131071  # K of an int8 product: 128 * 128 * K stays below 2^31
_HALF = (torch.float16, torch.bfloat16)

# The block's feed-forward branch keeps its activations in 8 bits when set (see feedforward_checkpoint8):
# 4.1 bytes per model-width element and layer instead of 14, for one rounding of the activations that the
# weight gradients and GELU's derivative read.  A training step of the 6-layer a1 model at 256 x 1024 tokens peaks at
# 22.6 GiB instead of 30.0 and takes 84 ms instead of 80.6 (its products run on this library's GEMM, which without
# checkpoints takes 88).  A branch whose modules have hooks, or a forward of their own, is called as modules, its
# activations in 16 bits.
FEEDFORWARD_CHECKPOINT8 = False


# ----------------------------------------------------------------------------- helpers
# A call on a few rows is over on the device in 2 to 4 us.  Tensors that lie as the kernels want them go through the
# _host_calls extension, which checks, allocates and launches in 4 to 6 us on the host; it answers None for anything
# else, and the functions here then copy, find the device or say what is wrong (8 to 16 us).
_host_module = None


class _NoHostCalls:
    """Stands for the extension where it is not built: leaves every call to the functions here."""

    def __getattr__(self, name: str):
        return lambda *args: None


def _host():
    global _host_module
    if _host_module is None:
        _lib.lib()
        try:
            from . import _host_calls
            built_for = getattr(_host_calls, "torch_version", "of unknown version")
            if built_for != torch.__version__:
                raise ImportError(f"built for PyTorch {built_for}, this is {torch.__version__}")
        except ImportError as error:
            warnings.warn(f"the _host_calls extension cannot be used ({error}): eight-bit calls take about 8 us longer on the "
                          "host; `python -m double_attention_b200.build` builds it", RuntimeWarning, stacklevel=3)
            _host_module = _NoHostCalls()
        else:
            _host_calls.set_check(_lib.check)
            _host_module = _host_calls
    return _host_module


_CODES = {torch.float16: _lib.DA_F16, torch.bfloat16: _lib.DA_BF16, torch.float32: _lib.DA_F32}


_entries: dict = {}  # bound entry points by name


def _launch(device: int, name: str, *args) -> None:
    """One library call on the current stream of CUDA device ``device``, whichever device is current."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(_lib.lib(), name)
    if device == torch._C._cuda_getDevice():
        status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _lib.check(name, status)


def _new(shape, dtype: torch.dtype, device: torch.device) -> Tensor:
    """A new dense tensor (torch.empty_strided takes 1.5 us on the host, torch.empty 2 to 4.5)."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _device_of(name: str, first: Tensor, *others: Tensor | None) -> int:
    device = first.get_device()
    if device < 0:
        raise ValueError(f"{name} requires CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name} requires its tensors on one device, got {first.device} and {t.device}")
    return device


def _float_code(name: str, what: str, t: Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} takes {what} in float32, bfloat16 or float16, got {t.dtype}")
    return code


def _half_code(name: str, what: str, t: Tensor) -> int:
    if t.dtype not in _HALF:
        raise ValueError(f"{name} takes {what} in bfloat16 or float16, got {t.dtype}")
    return _CODES[t.dtype]


def _inference_only(name: str, *tensors: Tensor | None) -> None:
    """Raises where a result would have to carry a gradient or a forward-mode tangent."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0 and forward_ad._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: call it on primal tensors")


def _rows(t: Tensor) -> tuple[Tensor, int, int]:
    """``(t, rows, row stride)`` of ``t`` [..., D] with unit column stride: as it lies, or a copy that has it."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // d, d
    if t.ndim != 2:
        t = t.reshape(-1, d)
    if t.stride(1) != 1 and d > 1:
        t = t.contiguous()
    return t, t.shape[0], t.stride(0)


def _round_up(n: int, to: int) -> int:
    return -(-n // to) * to


def _rows16(t: Tensor, elements: int) -> tuple[Tensor, int, int]:
    """As :func:`_rows`, every row on 16 bytes (``elements`` of them): as it lies, or copied to padded rows."""
    t, rows, stride = _rows(t)
    d = t.shape[-1]
    if not t.data_ptr() % 16:
        if not stride % elements and stride >= d:
            return t, rows, stride
        if rows == 1:  # has no stride of its own
            return t, rows, _round_up(d, elements)
    out = _new((rows, _round_up(d, elements)), t.dtype, t.device)
    out[:, :d] = t.reshape(rows, d)
    return out, rows, out.shape[1]


# ----------------------------------------------------------------------------- int8 rows
class Int8Rows(NamedTuple):
    """Rows in int8 with one scale each: ``values[..., k] * scale[...]``.

    values: int8 [..., K]; the operators here lay rows out on 16-byte boundaries (K rounded up), which the
    matrix product reads in place; other layouts are copied first.
    scale: fp32 [...].
    """

    values: Tensor
    scale: Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The values the rows stand for, each rounded once to ``dtype``."""
        name = "Int8Rows.dequantize"
        code = _CODES.get(dtype)
        if code is None:
            raise ValueError(f"{name} writes float32, bfloat16 or float16, got {dtype}")
        if self.values.is_cuda:
            out = _host().dequantize(self.values, self.scale, code)
            if out is not None:
                return out
        device = _check_rows(name, self)
        _inference_only(name, self.scale)
        out = _new(self.values.shape, dtype, self.values.device)
        if out.numel():
            q, rows, stride = _rows(self.values)
            d = q.shape[-1]
            _launch(device, "da_dequant_int8", q.data_ptr(), stride, self.scale.contiguous().data_ptr(), rows, d,
                    out.data_ptr(), code, d)
        return out


def _check_rows(name: str, x: Int8Rows) -> int:
    """The device of int8 rows, checked."""
    values, scale = x
    shape = values.shape
    if values.dtype != torch.int8 or not shape or not shape[-1]:
        raise ValueError(f"{name} takes int8 rows [..., K] with K at least 1, got {values.dtype} {tuple(shape)}")
    if scale.dtype != torch.float32 or scale.shape != shape[:-1]:
        raise ValueError(f"{name} takes one fp32 scale per row {tuple(shape[:-1])}, "
                         f"got {scale.dtype} {tuple(scale.shape)}")
    return _device_of(name, values, scale)


_QUANTIZE, _RMS, _LAYER = 0, 1, 2


def _norm_int8(name: str, x: Tensor, branch: Tensor | None, weight: Tensor | None, bias: Tensor | None, kind: int,
               eps: float) -> tuple[Tensor | None, Int8Rows]:
    if x.is_cuda:
        made = _host().norm(x, branch, weight, bias, kind, eps)
        if made is not None:
            return made[0], Int8Rows(made[1], made[2])
    device = _device_of(name, x, branch, weight, bias)
    shape = x.shape
    if not shape or not shape[-1]:
        raise ValueError(f"{name} takes rows [..., D] with D at least 1, got {tuple(shape)}")
    d = shape[-1]
    x_code = _float_code(name, "x", x)
    b_code = w_code = bias_code = 0
    if branch is not None:
        if branch.shape != shape:
            raise ValueError(f"branch shape {tuple(branch.shape)} does not match the residual {tuple(shape)}")
        b_code = _float_code(name, "the branch", branch)
    if weight is not None:
        w_code = _float_code(name, "weight", weight)
        weight = weight.contiguous()
        if bias is not None:
            bias_code = _float_code(name, "bias", bias)
            bias = bias.contiguous()
    _inference_only(name, x, branch, weight, bias)
    pitch = _round_up(d, 16)
    lead = shape[:-1]
    q = _new((*lead, pitch), torch.int8, x.device)
    scale = _new(lead, torch.float32, x.device)
    x2, rows, ldx = _rows(x)
    x_out, b2, ldb = None, None, 0
    if branch is not None:
        x_out = _new(shape, x.dtype, x.device)
        b2, _, ldb = _rows(branch)
    if rows:
        _launch(device, "da_norm_int8", x2.data_ptr(), x_code, ldx, ptr(b2), b_code, ldb, ptr(weight), w_code, ptr(bias),
                bias_code, kind, rows, d, eps, ptr(x_out), d, q.data_ptr(), pitch, scale.data_ptr())
    return x_out, Int8Rows(q if pitch == d else q[..., :d], scale)


def _rms_args(norm, x: Tensor) -> tuple[Tensor | None, float]:
    if not isinstance(norm, torch.nn.RMSNorm) or norm.normalized_shape != x.shape[-1:]:
        raise ValueError(f"expected an nn.RMSNorm over the last dimension of x {tuple(x.shape)}, got {norm}")
    # (without an eps of its own nn.RMSNorm takes that of the type it computes in, fp32 for all types here)
    return norm.weight, torch.finfo(torch.float32).eps if norm.eps is None else norm.eps


def _layer_args(norm, x: Tensor) -> tuple[Tensor | None, Tensor | None, float]:
    if not isinstance(norm, torch.nn.LayerNorm) or norm.normalized_shape != x.shape[-1:]:
        raise ValueError(f"expected an nn.LayerNorm over the last dimension of x {tuple(x.shape)}, got {norm}")
    return norm.weight, norm.bias, norm.eps


def rmsnorm_int8(x: Tensor, norm: torch.nn.RMSNorm) -> Int8Rows:
    """``norm(x)`` with its rows in int8: ``q = rint(y / scale)``, ``scale = max|y| / 127`` per row.

    x [..., D] in fp32, bf16 or fp16, any strides.  A row of zeros has scale 0; a row that holds a NaN or an
    infinity decodes to NaN throughout."""
    weight, eps = _rms_args(norm, x)
    return _norm_int8("rmsnorm_int8", x, None, weight, None, _RMS, eps)[1]


def add_rmsnorm_int8(x: Tensor, branch: Tensor, norm: torch.nn.RMSNorm) -> tuple[Tensor, Int8Rows]:
    """``(x + branch, norm(x + branch) in int8)`` in one pass; the sum keeps x's dtype and the norm reads it
    as rounded to that dtype."""
    weight, eps = _rms_args(norm, x)
    return _norm_int8("add_rmsnorm_int8", x, branch, weight, None, _RMS, eps)


def layernorm_int8(x: Tensor, norm: torch.nn.LayerNorm) -> Int8Rows:
    """:func:`rmsnorm_int8` for an ``nn.LayerNorm`` (the norm of this package's blocks)."""
    weight, bias, eps = _layer_args(norm, x)
    return _norm_int8("layernorm_int8", x, None, weight, bias, _LAYER, eps)[1]


def add_layernorm_int8(x: Tensor, branch: Tensor, norm: torch.nn.LayerNorm) -> tuple[Tensor, Int8Rows]:
    """:func:`add_rmsnorm_int8` for an ``nn.LayerNorm``."""
    weight, bias, eps = _layer_args(norm, x)
    return _norm_int8("add_layernorm_int8", x, branch, weight, bias, _LAYER, eps)


def quantize_int8(x: Tensor) -> Int8Rows:
    """Rows of ``x`` [..., D] in int8 with one scale each: a Linear's weight [N, K] once (a scale per output
    channel), or activations on their way into :func:`int8_linear` (a scale per token)."""
    return _norm_int8("quantize_int8", x, None, None, None, _QUANTIZE, 0.0)[1]


# ----------------------------------------------------------------------------- int8 matrix product
def int8_linear(x: Int8Rows, weight: Int8Rows, bias: Tensor | None = None, *, gelu: bool = False,
                dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``y[..., n] = sum_k x[..., k] weight[n, k] (+ bias[n])``, through GELU when asked, from int8 rows.

    The sum over K (at most 131071) is exact; it is scaled, biased and activated in fp32 and rounded once to
    ``dtype`` (bf16, fp16 or fp32).  x [..., K], weight [N, K], bias [N] in any float dtype."""
    name = "int8_linear"
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"{name} writes float32, bfloat16 or float16, got {dtype}")
    if x.values.is_cuda:
        out = _host().linear(x.values, x.scale, weight.values, weight.scale, bias, gelu, code,
                             ops.workspace(x.values.device).status)
        if out is not None:
            return out
    device = _check_rows(name, x)
    w_shape = weight.values.shape
    if _check_rows(name, weight) != device or len(w_shape) != 2:
        raise ValueError(f"{name} takes a weight [N, K] on x's device, got {tuple(w_shape)} on {weight.values.device}")
    n, k = w_shape
    if x.values.shape[-1] != k or k > MAX_INNER or n < 1:
        raise ValueError(f"{name}: x {tuple(x.values.shape)} and weight {tuple(w_shape)} must share "
                         f"an inner size of 1 to {MAX_INNER}")
    bias_ptr, bias_code = None, 0
    if bias is not None:
        bias_code = _float_code(name, "a bias", bias)
        if bias.shape != (n,) or bias.get_device() != device:
            raise ValueError(f"{name} takes a bias of shape [{n}] on x's device, got {tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    _inference_only(name, x.scale, weight.scale, bias)
    out = _new((*x.values.shape[:-1], n), dtype, x.values.device)
    xq, rows, ldx = _rows16(x.values, 16)
    if rows:
        wq, _, ldw = _rows16(weight.values, 16)
        xs, ws = x.scale.contiguous(), weight.scale.contiguous()
        _launch(device, "da_gemm_i8", xq.data_ptr(), ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), bias_ptr,
                bias_code, int(gelu), out.data_ptr(), n, code, rows, n, k,
                ops.workspace(out.device).status.data_ptr())
    return out


# ----------------------------------------------------------------------------- checkpoints
@dataclass(frozen=True)
class Checkpoint8:
    """An activation kept in 8 bits: ``values * 2^exponent``, an exponent per 32 columns of a row.

    values: int8 [rows, ceil(D / 32) * 32], columns past D zero;  exponent: int8 [rows, ceil(D / 32)], -128
    marking a block that held a NaN or an infinity (it restores to NaN).  shape and dtype are the
    activation's; the values it stands for are exact in that dtype."""

    values: Tensor
    exponent: Tensor
    shape: tuple[int, ...]
    dtype: torch.dtype

    @property
    def rows(self) -> int:
        return self.values.shape[0]

    def restore(self) -> Tensor:
        """The values the checkpoint stands for, in the activation's shape and dtype."""
        device = _check_checkpoint("Checkpoint8.restore", self)
        out = _new(self.shape, self.dtype, self.values.device)
        if out.numel():
            d = self.shape[-1]
            _launch(device, "da_checkpoint8_restore", self.values.data_ptr(), self.exponent.data_ptr(), self.rows, d,
                    out.data_ptr(), _CODES[self.dtype], d)
        return out


def _check_checkpoint(name: str, c: Checkpoint8) -> int:
    """The device of a checkpoint, checked."""
    values, exponent, shape = c.values, c.exponent, c.shape
    d = shape[-1] if shape else 0
    blocks = -(-d // BLOCK)
    rows = math.prod(shape[:-1])
    if (c.dtype not in _HALF or d < 1 or values.dtype != torch.int8 or exponent.dtype != torch.int8
            or values.shape != (rows, blocks * BLOCK) or exponent.shape != (rows, blocks)
            or not values.is_contiguous() or not exponent.is_contiguous() or values.data_ptr() % 16):
        raise ValueError(f"{name} takes a checkpoint of a 16-bit activation: dense int8 values "
                         f"[{rows}, {blocks * BLOCK}] on 16 bytes and exponents [{rows}, {blocks}], got {c.dtype} "
                         f"{tuple(values.shape)}, {tuple(exponent.shape)}")
    return _device_of(name, values, exponent)


def _checkpoint8(name: str, x: Tensor, gelu: bool) -> tuple[Tensor | None, Checkpoint8]:
    if x.is_cuda:
        made = _host().checkpoint(x, gelu)
        if made is not None:
            return made[0], Checkpoint8(made[1], made[2], tuple(x.shape), x.dtype)
    device = _device_of(name, x)
    code = _half_code(name, "an activation", x)
    shape = x.shape
    if not shape or not shape[-1]:
        raise ValueError(f"{name} takes rows [..., D] with D at least 1, got {tuple(shape)}")
    x2, rows, ldx = _rows(x)
    d = shape[-1]
    blocks = -(-d // BLOCK)
    values = _new((rows, blocks * BLOCK), torch.int8, x.device)
    exponent = _new((rows, blocks), torch.int8, x.device)
    h = _new(shape, x.dtype, x.device) if gelu else None
    if rows:
        _launch(device, "da_checkpoint8", x2.data_ptr(), code, ldx, rows, d, int(gelu), ptr(h), d, values.data_ptr(),
                exponent.data_ptr())
    return h, Checkpoint8(values, exponent, tuple(shape), x.dtype)


def checkpoint8(x: Tensor) -> Checkpoint8:
    """``x`` [..., D] (fp16 or bf16) in 8 bits.  Not differentiable itself: see :func:`linear_checkpoint8`."""
    _inference_only("checkpoint8", x)
    return _checkpoint8("checkpoint8", x, False)[1]


def gelu_checkpoint8(z: Tensor) -> tuple[Tensor, Checkpoint8]:
    """``(GELU(z), z in 8 bits)`` in one pass (the exact erf form of GELU, as nn.GELU's default)."""
    _inference_only("gelu_checkpoint8", z)
    return _checkpoint8("gelu_checkpoint8", z, True)


def gelu_checkpoint8_backward(dh: Tensor, kept: Checkpoint8) -> tuple[Tensor, Tensor]:
    """``(dh * GELU'(z), GELU(z))`` with z as kept: the gradient of GELU's input, and its output once more for
    the next layer's weight gradient."""
    name = "gelu_checkpoint8_backward"
    if dh.is_cuda and dh.shape == kept.shape and dh.dtype == kept.dtype:
        made = _host().gelu_backward(dh, kept.values, kept.exponent)
        if made is not None:
            return made
    device = _check_checkpoint(name, kept)
    if dh.shape != kept.shape or dh.dtype != kept.dtype or dh.get_device() != device:
        raise ValueError(f"{name}: dh {dh.dtype} {tuple(dh.shape)} on {dh.device} does not match the checkpoint "
                         f"{kept.dtype} {kept.shape} on {kept.values.device}")
    _inference_only(name, dh)
    dz = _new(kept.shape, dh.dtype, dh.device)
    h = _new(kept.shape, dh.dtype, dh.device)
    d2, rows, ldd = _rows(dh)
    if rows:
        d = kept.shape[-1]
        _launch(device, "da_checkpoint8_gelu_bwd", d2.data_ptr(), _CODES[dh.dtype], ldd, kept.values.data_ptr(),
                kept.exponent.data_ptr(), rows, d, dz.data_ptr(), d, h.data_ptr(), d)
    return dz, h


def weight_grad_checkpoint8(dy: Tensor, kept: Checkpoint8, dtype: torch.dtype | None = None) -> Tensor:
    """dW [N, K] = sum over the rows of dy [..., N]^T x [..., K], x as kept: a Linear's weight gradient,
    accumulated in fp32 in a fixed order (bit-reproducible) and stored in ``dtype`` (dy's, the default, or
    fp32)."""
    name = "weight_grad_checkpoint8"
    shape, dtype = dy.shape, dtype or dy.dtype
    if (kept.shape and shape[:-1] == kept.shape[:-1] and dy.dtype == kept.dtype and dtype in (torch.float32, dy.dtype) and dy.is_cuda):
        made = _host().weight_grad(dy, kept.values, kept.exponent, kept.shape[-1], _CODES[dtype],
                                   ops.workspace(dy.device).status)
        if made is not None:
            return made
    device = _check_checkpoint(name, kept)
    if not shape or shape[:-1] != kept.shape[:-1] or not shape[-1] or dy.dtype != kept.dtype or dy.get_device() != device:
        raise ValueError(f"{name}: dy {dy.dtype} {tuple(shape)} on {dy.device} does not match the checkpoint "
                         f"{kept.dtype} {kept.shape} on {kept.values.device}")
    if dtype != torch.float32 and dtype != dy.dtype:
        raise ValueError(f"{name} stores fp32 or dy's {dy.dtype}, got {dtype}")
    _inference_only(name, dy)
    n, k = shape[-1], kept.shape[-1]
    out = _new((n, k), dtype, dy.device)
    d2, rows, ldd = _rows16(dy, 8) if n % 8 == 0 else _rows(dy)
    if not rows:
        return out.zero_()
    if ldd < n:  # (one row, or rows that share their values)
        d2, ldd = d2.contiguous(), n
    elems = _lib.lib().da_checkpoint8_wgrad_workspace_elems(rows, n, k)
    work = _new((elems,), torch.float32, dy.device) if elems else None
    _launch(device, "da_checkpoint8_wgrad", d2.data_ptr(), _CODES[dy.dtype], ldd, kept.values.data_ptr(),
            kept.exponent.data_ptr(), rows, n, k, out.data_ptr(), _CODES[dtype], k, ptr(work), elems,
            ops.workspace(out.device).status.data_ptr())
    return out


class _FirstOrder(torch.autograd.Function):
    """A gradient as it is; differentiated again (it depends on dout, on what was kept and on the weights), it raises."""

    @staticmethod
    def forward(ctx, grad: Tensor, dout: Tensor, name: str):  # type: ignore[override]
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):  # type: ignore[override]
        raise RuntimeError(f"{ctx.name} has no second derivative")


def _first_order(name: str):
    """A Function's backward that runs outside any graph; under create_graph=True its results raise when differentiated."""

    def of(backward):
        def wrapped(ctx, dout: Tensor):
            with torch.no_grad():
                grads = backward(ctx, dout)
            if not torch.is_grad_enabled():
                return grads
            return tuple(None if g is None else _FirstOrder.apply(g.detach().requires_grad_(), dout, name) for g in grads)

        return wrapped

    return of


class _LinearCheckpoint8(torch.autograd.Function):
    """y = x W^T (+ b) on the tcgen05 GEMM; x is kept for dW in 8 bits."""

    @staticmethod
    def forward(ctx, x2d: Tensor, weight: Tensor, bias: Tensor | None, dtype: torch.dtype):  # type: ignore[override]
        w = weight.to(dtype)
        out = torch.empty(x2d.shape[0], w.shape[0], dtype=dtype, device=x2d.device)
        ops.gemm_ex(x2d, w, False, out, bias=None if bias is None else bias.to(dtype))
        kept = _checkpoint8("linear_checkpoint8", x2d, False)[1] if ctx.needs_input_grad[1] else None
        ctx.save_for_backward(w, *(() if kept is None else (kept.values, kept.exponent)))
        ctx.meta = (tuple(x2d.shape), dtype, weight.dtype, None if bias is None else bias.dtype)
        return out

    @staticmethod
    @_first_order("linear_checkpoint8")
    def backward(ctx, dout: Tensor):  # type: ignore[override]
        w, *kept = ctx.saved_tensors
        shape, dtype, weight_dtype, bias_dtype = ctx.meta
        need = ctx.needs_input_grad
        dout = dout.to(dtype).contiguous()
        dx = dw = db = None
        if need[0]:
            dx = torch.empty(shape, dtype=dtype, device=w.device)
            ops.gemm_ex(dout, w, True, dx)
        if need[1]:
            dw = _weight_grad_as(dout, Checkpoint8(*kept, shape, dtype), weight_dtype)
        if need[2]:
            db = ops._bias_grad(dout).to(bias_dtype)
        return dx, dw, db, None


def _weight_grad_as(dy: Tensor, kept: Checkpoint8, dtype: torch.dtype) -> Tensor:
    store = dtype if dtype == dy.dtype else torch.float32
    return weight_grad_checkpoint8(dy, kept, store).to(dtype)


class _FeedForwardCheckpoint8(torch.autograd.Function):
    """second(GELU(first(x))) on the tcgen05 GEMM; x (for dW1 alone) and the pre-activation z are kept in 8 bits, the
    hidden activation not at all (the backward rebuilds it from z)."""

    @staticmethod
    def forward(ctx, x2d: Tensor, w1: Tensor, b1: Tensor | None, w2: Tensor, b2: Tensor | None,  # type: ignore[override]
                dtype: torch.dtype):
        m = x2d.shape[0]
        w1c, w2c = w1.to(dtype), w2.to(dtype)
        z = torch.empty(m, w1c.shape[0], dtype=dtype, device=x2d.device)
        ops.gemm_ex(x2d, w1c, False, z, bias=None if b1 is None else b1.to(dtype))
        h, zk = _checkpoint8("feedforward_checkpoint8", z, True)
        out = torch.empty(m, w2c.shape[0], dtype=dtype, device=x2d.device)
        ops.gemm_ex(h, w2c, False, out, bias=None if b2 is None else b2.to(dtype))
        xk = _checkpoint8("feedforward_checkpoint8", x2d, False)[1] if ctx.needs_input_grad[1] else None
        ctx.save_for_backward(w1c, w2c, zk.values, zk.exponent, *(() if xk is None else (xk.values, xk.exponent)))
        ctx.meta = (tuple(x2d.shape), zk.shape, dtype)
        ctx.param_dtypes = tuple(None if p is None else p.dtype for p in (w1, b1, w2, b2))
        return out

    @staticmethod
    @_first_order("feedforward_checkpoint8")
    def backward(ctx, dout: Tensor):  # type: ignore[override]
        w1c, w2c, zv, ze, *xk = ctx.saved_tensors
        x_shape, z_shape, dtype = ctx.meta
        need, pd = ctx.needs_input_grad, ctx.param_dtypes
        dout = dout.to(dtype).contiguous()
        dx = dw1 = db1 = dw2 = db2 = None
        dh = torch.empty(z_shape, dtype=dtype, device=dout.device)
        ops.gemm_ex(dout, w2c, True, dh)  # dH = dOut . W2
        dz, h = gelu_checkpoint8_backward(dh, Checkpoint8(zv, ze, z_shape, dtype))
        if need[3]:
            dw2 = ops.weight_grad(dout, h, w2c.shape[0], w2c.shape[1], x_shape[0], pd[2])  # dW2 = dOut^T . h
        if need[4]:
            db2 = ops._bias_grad(dout).to(pd[3])
        if need[1]:
            dw1 = _weight_grad_as(dz, Checkpoint8(*xk, x_shape, dtype), pd[0])  # dW1 = dZ^T . x
        if need[2]:
            db1 = ops._bias_grad(dz).to(pd[1])
        if need[0]:
            dx = torch.empty(x_shape, dtype=dtype, device=dout.device)
            ops.gemm_ex(dz, w1c, True, dx)  # dX = dZ . W1
        return dx, dw1, db1, dw2, db2, None


def _linear_rows(x: Tensor) -> tuple[Tensor, torch.dtype]:
    dtype = ops._linear_dtype(x)
    x2d = x.reshape(-1, x.shape[-1]).to(dtype)
    return (x2d if x2d.is_contiguous() else x2d.contiguous()), dtype


def own_forward(module: torch.nn.Module, kind: type) -> bool:
    """Whether ``module`` computes something else than ``kind`` does (a subclass, or a forward set on it)."""
    return type(module).forward is not kind.forward or "forward" in vars(module)


def is_plain(module: torch.nn.Module, kind: type) -> bool:
    """Whether calling ``module`` runs ``kind``'s forward and nothing else: no forward of its own, no hooks."""
    return not (own_forward(module, kind) or module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks or torch.nn.modules.module._has_any_global_hook())


def checkpoint8_supported(x: Tensor, *layers: torch.nn.Linear) -> bool:
    """Whether :func:`linear_checkpoint8` / :func:`feedforward_checkpoint8` cover these layers on ``x``:
    half-precision compute on CUDA, widths multiples of 128."""
    return all(ops.linear_supported(x, n) and n.in_features % 128 == 0 for n in layers)


def linear_checkpoint8(x: Tensor, layer: torch.nn.Linear) -> Tensor:
    """``layer(x)`` as :func:`ops.linear` computes it, the input kept for the weight gradient in 8 bits."""
    if not checkpoint8_supported(x, layer):
        raise NotImplementedError("linear_checkpoint8 needs half-precision compute on CUDA and widths divisible by 128")
    x2d, dtype = _linear_rows(x)
    out = _LinearCheckpoint8.apply(x2d, layer.weight, layer.bias, dtype)
    return out.view(*x.shape[:-1], out.shape[-1])


def feedforward_checkpoint8(x: Tensor, first: torch.nn.Linear, second: torch.nn.Linear) -> Tensor:
    """``second(GELU(first(x)))`` as :func:`ops.feedforward` computes it; what the backward keeps of x and of
    the pre-activation takes 8 bits an element, and the hidden activation is rebuilt."""
    if not (checkpoint8_supported(x, first, second) and first.out_features == second.in_features):
        raise NotImplementedError("feedforward_checkpoint8 needs half-precision compute on CUDA and widths divisible "
                                  "by 128")
    x2d, dtype = _linear_rows(x)
    out = _FeedForwardCheckpoint8.apply(x2d, first.weight, first.bias, second.weight, second.bias, dtype)
    return out.view(*x.shape[:-1], out.shape[-1])
