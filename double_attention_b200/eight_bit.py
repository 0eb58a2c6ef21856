"""Eight-bit operators: an int8 serving path and 8-bit activation checkpoints for training.

Serving.  A norm leaves its rows in int8 with one scale per token (:func:`add_rmsnorm_int8`,
:func:`add_layernorm_int8` and their forms without a branch), activations that no norm precedes go
through :func:`quantize_int8` -- as do the weights, once, with one scale per output channel -- and
:func:`int8_linear` multiplies the two on the int8 tensor cores, from a single token to long batches.
These operators have no backward; called on tensors that require a gradient they raise.

Training.  :func:`gelu_checkpoint8` keeps GELU's input in 8 bits (blocks of 32 columns sharing a
power-of-two scale) in place of the 16-bit tensor, :func:`gelu_checkpoint8_backward` and
:func:`weight_grad_checkpoint8` work from such a checkpoint, and :func:`linear_checkpoint8` and
:func:`feedforward_checkpoint8` put them together behind autograd: a Linear and the block's
feed-forward branch whose saved activations take 8 bits an element.

Every numeric step runs in the kernels of ``libda_b200.so``; unsupported inputs raise.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib, ops
from ._lib import call, dtype_code, ptr, stream_ptr

BLOCK = 32          # columns of a checkpoint that share one exponent
MAX_INNER = 131071  # K of an int8 product: 128 * 128 * K stays below 2^31
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_HALF = (torch.float16, torch.bfloat16)

# The block's feed-forward branch keeps its activations in 8 bits when set (see feedforward_checkpoint8):
# 4.1 bytes per model-width element and layer instead of 14, for one rounding of the activations that the
# weight gradients and GELU's derivative read.
FEEDFORWARD_CHECKPOINT8 = False


# ----------------------------------------------------------------------------- helpers
def _launch(device: torch.device, name: str, *args) -> None:
    """One library call on ``device``'s current stream, whichever device is current."""
    if device.index == torch.cuda.current_device():
        call(name, *args, stream_ptr(device))
    else:
        with torch.cuda.device(device):
            call(name, *args, stream_ptr(device))


def _check_cuda(name: str, first: Tensor, *others: Tensor | None) -> torch.device:
    if not first.is_cuda:
        raise ValueError(f"{name} requires CUDA tensors")
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{name} requires its tensors on one device, got {device} and {t.device}")
    return device


def _check_float(name: str, what: str, t: Tensor, allowed=_FLOATS) -> None:
    if t.dtype not in allowed:
        names = ", ".join(str(d).removeprefix("torch.") for d in allowed)
        raise ValueError(f"{name} takes {what} in {names}, got {t.dtype}")


def _inference_only(name: str, *tensors: Tensor | None) -> None:
    if ops._grad_wanted(*tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() or on detached tensors")


def _rows(t: Tensor) -> Tensor:
    """``t`` [..., D] as [rows, D] with unit column stride; a view where its strides allow one."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _round_up(n: int, to: int) -> int:
    return -(-n // to) * to


def _aligned_rows(t: Tensor, elements: int) -> Tensor:
    """[rows, D] with rows starting on 16 bytes (``elements`` of them): as is, or copied to padded rows."""
    rows, d = t.shape
    stride = t.stride(0)
    if t.data_ptr() % 16 == 0 and (rows == 1 or (stride >= d and stride % elements == 0)):
        return t
    out = torch.empty(rows, _round_up(d, elements), dtype=t.dtype, device=t.device)[:, :d]
    return out.copy_(t)


def _stride16(t: Tensor, elements: int) -> int:
    """The row stride handed to a kernel that wants 16-byte rows (a single row has none of its own)."""
    return t.stride(0) if t.shape[0] > 1 else _round_up(t.shape[1], elements)


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
        q, scale = _check_rows("Int8Rows.dequantize", self)
        if dtype not in _FLOATS:
            raise ValueError(f"Int8Rows.dequantize writes float32, bfloat16 or float16, got {dtype}")
        out = torch.empty(self.values.shape, dtype=dtype, device=q.device)
        if out.numel():
            rows, d = q.shape
            _launch(q.device, "da_dequant_int8", q.data_ptr(), q.stride(0), scale.data_ptr(), rows, d,
                    out.data_ptr(), dtype_code(dtype), d)
        return out


def _check_rows(name: str, x: Int8Rows) -> tuple[Tensor, Tensor]:
    """``(values [rows, K], scale [rows])`` of int8 rows, checked."""
    values, scale = x
    if values.dtype != torch.int8 or values.ndim < 1:
        raise ValueError(f"{name} takes int8 rows [..., K], got {values.dtype} {tuple(values.shape)}")
    if scale.dtype != torch.float32 or scale.shape != values.shape[:-1]:
        raise ValueError(f"{name} takes one fp32 scale per row {tuple(values.shape[:-1])}, "
                         f"got {scale.dtype} {tuple(scale.shape)}")
    _check_cuda(name, values, scale)
    if scale.ndim != 1:
        scale = scale.reshape(-1)
    return _rows(values), scale if scale.is_contiguous() else scale.contiguous()


_QUANTIZE, _RMS, _LAYER = 0, 1, 2


def _norm_int8(name: str, x: Tensor, branch: Tensor | None, weight: Tensor | None, bias: Tensor | None, kind: int,
               eps: float) -> tuple[Tensor | None, Int8Rows]:
    device = _check_cuda(name, x, branch, weight, bias)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} takes rows [..., D] with D at least 1, got {tuple(x.shape)}")
    d = x.shape[-1]
    _check_float(name, "x", x)
    if branch is not None:
        if branch.shape != x.shape:
            raise ValueError(f"branch shape {tuple(branch.shape)} does not match the residual {tuple(x.shape)}")
        _check_float(name, "the branch", branch)
    for what, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_float(name, what, t)
            if t.shape != (d,):
                raise ValueError(f"{name} takes a {what} of shape [{d}], got {tuple(t.shape)}")
    _inference_only(name, x, branch, weight, bias)
    lead = x.shape[:-1]
    x2 = _rows(x)
    rows = x2.shape[0]
    x_out = b2 = None
    if branch is not None:
        b2 = _rows(branch)
        x_out = torch.empty(x.shape, dtype=x.dtype, device=device)
    pitch = _round_up(d, 16)
    q = torch.empty(rows, pitch, dtype=torch.int8, device=device)
    scale = torch.empty(lead, dtype=torch.float32, device=device)
    if rows:
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        _launch(device, "da_norm_int8", x2.data_ptr(), dtype_code(x.dtype), x2.stride(0), ptr(b2),
                0 if b2 is None else dtype_code(b2.dtype), 0 if b2 is None else b2.stride(0), ptr(w),
                0 if w is None else dtype_code(w.dtype), ptr(b), 0 if b is None else dtype_code(b.dtype), kind, rows, d,
                eps, ptr(x_out), d, q.data_ptr(), pitch, scale.data_ptr())
    if pitch != d:
        q = q[:, :d]
    if len(lead) != 1:
        q = q.unflatten(0, lead) if lead else q[0]
    return x_out, Int8Rows(q, scale)


def _rms_args(norm, x: Tensor) -> tuple[Tensor | None, float]:
    if not isinstance(norm, torch.nn.RMSNorm) or tuple(norm.normalized_shape) != (x.shape[-1],):
        raise ValueError(f"expected an nn.RMSNorm over the last dimension of x ({x.shape[-1]}), got {norm}")
    return norm.weight, torch.finfo(x.dtype).eps if norm.eps is None else norm.eps


def _layer_args(norm, x: Tensor) -> tuple[Tensor | None, Tensor | None, float]:
    if not isinstance(norm, torch.nn.LayerNorm) or tuple(norm.normalized_shape) != (x.shape[-1],):
        raise ValueError(f"expected an nn.LayerNorm over the last dimension of x ({x.shape[-1]}), got {norm}")
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
    xq, xs = _check_rows(name, x)
    wq, ws = _check_rows(name, weight)
    if weight.values.ndim != 2:
        raise ValueError(f"{name} takes a weight [N, K], got {tuple(weight.values.shape)}")
    n, k = wq.shape
    device = _check_cuda(name, xq, wq, bias)
    if xq.shape[1] != k or not 0 < k <= MAX_INNER or n < 1:
        raise ValueError(f"{name}: x {tuple(x.values.shape)} and weight {tuple(weight.values.shape)} must share "
                         f"an inner size of 1 to {MAX_INNER}")
    if dtype not in _FLOATS:
        raise ValueError(f"{name} writes float32, bfloat16 or float16, got {dtype}")
    bias_code = 0
    if bias is not None:
        _check_float(name, "a bias", bias)
        if bias.shape != (n,):
            raise ValueError(f"{name} takes a bias of shape [{n}], got {tuple(bias.shape)}")
        _inference_only(name, bias)
        bias = bias.contiguous()
        bias_code = dtype_code(bias.dtype)
    lead = x.values.shape[:-1]
    out = torch.empty(*lead, n, dtype=dtype, device=device)
    rows = xq.shape[0]
    if rows:
        xq, wq = _aligned_rows(xq, 16), _aligned_rows(wq, 16)
        _launch(device, "da_gemm_i8", xq.data_ptr(), _stride16(xq, 16), xs.data_ptr(), wq.data_ptr(), _stride16(wq, 16),
                ws.data_ptr(), ptr(bias), bias_code, int(gelu), out.data_ptr(), n, dtype_code(dtype), rows, n, k,
                ops.workspace(device).status.data_ptr())
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
        out = torch.empty(self.shape, dtype=self.dtype, device=device)
        if out.numel():
            d = self.shape[-1]
            _launch(device, "da_checkpoint8_restore", self.values.data_ptr(), self.exponent.data_ptr(), self.rows, d,
                    out.data_ptr(), dtype_code(self.dtype), d)
        return out


def _check_checkpoint(name: str, c: Checkpoint8) -> torch.device:
    d = c.shape[-1]
    blocks = -(-d // BLOCK)
    rows = 1
    for s in c.shape[:-1]:
        rows *= s
    if (c.dtype not in _HALF or d < 1 or c.values.dtype != torch.int8 or c.exponent.dtype != torch.int8
            or c.values.shape != (rows, blocks * BLOCK) or c.exponent.shape != (rows, blocks)
            or not c.values.is_contiguous() or not c.exponent.is_contiguous() or c.values.data_ptr() % 16):
        raise ValueError(f"{name} takes a checkpoint of a 16-bit activation: dense int8 values "
                         f"[{rows}, {blocks * BLOCK}] and exponents [{rows}, {blocks}], got {c.dtype} "
                         f"{tuple(c.values.shape)}, {tuple(c.exponent.shape)}")
    return _check_cuda(name, c.values, c.exponent)


def _checkpoint8(name: str, x: Tensor, gelu: bool) -> tuple[Tensor | None, Checkpoint8]:
    device = _check_cuda(name, x)
    _check_float(name, "an activation", x, _HALF)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} takes rows [..., D] with D at least 1, got {tuple(x.shape)}")
    x2 = _rows(x)
    rows, d = x2.shape
    blocks = -(-d // BLOCK)
    values = torch.empty(rows, blocks * BLOCK, dtype=torch.int8, device=device)
    exponent = torch.empty(rows, blocks, dtype=torch.int8, device=device)
    h = torch.empty(x.shape, dtype=x.dtype, device=device) if gelu else None
    if rows:
        _launch(device, "da_checkpoint8", x2.data_ptr(), dtype_code(x.dtype), x2.stride(0), rows, d, int(gelu), ptr(h), d,
                values.data_ptr(), exponent.data_ptr())
    return h, Checkpoint8(values, exponent, tuple(x.shape), x.dtype)


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
    device = _check_checkpoint(name, kept)
    _check_cuda(name, kept.values, dh)
    if tuple(dh.shape) != kept.shape or dh.dtype != kept.dtype:
        raise ValueError(f"{name}: dh {dh.dtype} {tuple(dh.shape)} does not match the checkpoint {kept.dtype} {kept.shape}")
    _inference_only(name, dh)
    dz = torch.empty(kept.shape, dtype=dh.dtype, device=device)
    h = torch.empty(kept.shape, dtype=dh.dtype, device=device)
    if dz.numel():
        d2 = _rows(dh)
        rows, d = d2.shape
        _launch(device, "da_checkpoint8_gelu_bwd", d2.data_ptr(), dtype_code(dh.dtype), d2.stride(0), kept.values.data_ptr(),
                kept.exponent.data_ptr(), rows, d, dz.data_ptr(), d, h.data_ptr(), d)
    return dz, h


def weight_grad_checkpoint8(dy: Tensor, kept: Checkpoint8, dtype: torch.dtype | None = None) -> Tensor:
    """dW [N, K] = sum over the rows of dy [..., N]^T x [..., K], x as kept: a Linear's weight gradient,
    accumulated in fp32 in a fixed order (bit-reproducible) and stored in ``dtype`` (dy's, the default, or
    fp32)."""
    name = "weight_grad_checkpoint8"
    device = _check_checkpoint(name, kept)
    _check_cuda(name, kept.values, dy)
    if tuple(dy.shape[:-1]) != kept.shape[:-1] or dy.dtype != kept.dtype or dy.shape[-1] < 1:
        raise ValueError(f"{name}: dy {dy.dtype} {tuple(dy.shape)} does not match the checkpoint {kept.dtype} {kept.shape}")
    dtype = dtype or dy.dtype
    if dtype not in (torch.float32, dy.dtype):
        raise ValueError(f"{name} stores fp32 or dy's {dy.dtype}, got {dtype}")
    _inference_only(name, dy)
    n, k = dy.shape[-1], kept.shape[-1]
    out = torch.empty(n, k, dtype=dtype, device=device)
    d2 = _rows(dy)
    rows = d2.shape[0]
    if not rows:
        return out.zero_()
    d2 = _aligned_rows(d2, 8)
    elems = int(_lib.lib().da_checkpoint8_wgrad_workspace_elems(rows, n, k))
    work = torch.empty(max(elems, 4), dtype=torch.float32, device=device)
    _launch(device, "da_checkpoint8_wgrad", d2.data_ptr(), dtype_code(dy.dtype), _stride16(d2, 8), kept.values.data_ptr(),
            kept.exponent.data_ptr(), rows, n, k, out.data_ptr(), dtype_code(dtype), k, work.data_ptr(), work.numel(),
            ops.workspace(device).status.data_ptr())
    return out


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
    """second(GELU(first(x))) on the tcgen05 GEMM; x and the pre-activation z are kept in 8 bits, the hidden
    activation not at all (the backward rebuilds it from z)."""

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
        xk = _checkpoint8("feedforward_checkpoint8", x2d, False)[1]
        ctx.save_for_backward(w1c, w2c, xk.values, xk.exponent, zk.values, zk.exponent)
        ctx.meta = (xk.shape, zk.shape, dtype)
        ctx.param_dtypes = tuple(None if p is None else p.dtype for p in (w1, b1, w2, b2))
        return out

    @staticmethod
    def backward(ctx, dout: Tensor):  # type: ignore[override]
        w1c, w2c, xv, xe, zv, ze = ctx.saved_tensors
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
            dw1 = _weight_grad_as(dz, Checkpoint8(xv, xe, x_shape, dtype), pd[0])  # dW1 = dZ^T . x
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
