"""The C-ABI library loads on a CPU-only host and exports every entry point
declared in include/*.h; no compute is called here."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from double_attention_b200 import _lib

REPO = Path(__file__).resolve().parent.parent


def declared_symbols() -> list[str]:
    names = []
    for header in sorted((REPO / "include").glob("*.h")):
        names += re.findall(r"^DA_API\s+[\w\s\*]+?\b(da_\w+)\s*\(", header.read_text(), flags=re.M)
    return names


def test_header_declares_entry_points() -> None:
    names = declared_symbols()
    for required in ("da_dict_norm_fwd", "da_route_fwd", "da_attn_fwd", "da_gemm", "da_status_string"):
        assert required in names


def test_library_loads_and_exports_every_declared_symbol() -> None:
    handle = _lib.lib()
    for name in declared_symbols():
        assert hasattr(handle, name), name
    assert b"sm_100a" in handle.da_version()
    assert handle.da_status_string(_lib.DA_ERR_SHAPE) == b"unsupported or inconsistent shape"
    assert _lib.kernel_launches() >= 0


def test_bound_signatures_cover_compute_entry_points() -> None:
    for name in declared_symbols():
        if name in ("da_version", "da_status_string", "da_last_cuda_error", "da_kernel_launches"):
            continue
        assert name in _lib.SIGNATURES, f"{name} has no ctypes signature"


def test_argument_validation_happens_before_any_device_work() -> None:
    handle = _lib.lib()
    # null pointers are rejected on the host (no CUDA call is made)
    assert handle.da_route_fwd(*([None] * 1), *([0] * 8), *([None] * 4), ctypes.c_float(1e-6), 1, 1,
                               *([None] * 5), 0, None, None) == _lib.DA_ERR_NULL
    with pytest.raises(ValueError):
        _lib.check("da_gemm", _lib.DA_ERR_SHAPE)
    with pytest.raises(NotImplementedError):
        _lib.check("da_attn_fwd", _lib.DA_ERR_UNSUPPORTED)


def test_layernorm_entry_points_validate_on_the_host() -> None:
    handle = _lib.lib()
    f32 = ctypes.c_float(1e-5)
    # a null input, then an unsupported width: both refused before any CUDA call
    assert handle.da_add_layernorm_fwd(None, None, 0, None, None, 8, 512, f32, None, None, 1, None, None,
                                       None) == _lib.DA_ERR_NULL
    buf = (ctypes.c_float * 4096)()
    p = ctypes.addressof(buf)
    assert handle.da_add_layernorm_fwd(p, None, 0, p, p, 8, 500, f32, None, p, 1, p, p, None) == _lib.DA_ERR_SHAPE
    assert handle.da_add_layernorm_fwd(p, None, 0, p, p, 8, 512, f32, None, p, 7, p, p, None) == _lib.DA_ERR_DTYPE
    # the backward's partial-sum buffer must have the queried number of blocks
    blocks = handle.da_layernorm_bwd_blocks(1)
    assert blocks == 1
    assert handle.da_add_layernorm_bwd(p, 1, None, p, p, p, p, 1, 512, p, None, 0, p, blocks + 1, None, None,
                                       None) == _lib.DA_ERR_WORKSPACE


def test_fused_norms_only_for_cuda_fp32_rows() -> None:
    import torch
    import torch.nn as nn

    from double_attention_b200 import ops

    norm = nn.LayerNorm(512)
    assert not ops.layernorm_supported(torch.zeros(2, 512), norm)            # CPU tensor: plain nn.LayerNorm
    assert not ops.layernorm_supported(torch.zeros(2, 500), nn.LayerNorm(500))


def test_eight_bit_entry_points_validate_on_the_host() -> None:
    handle = _lib.lib()
    eps = ctypes.c_float(1e-6)
    raw = (ctypes.c_float * 4096)()
    p = (ctypes.addressof(raw) + 63) // 64 * 64

    def norm(x=p, x_dtype=2, branch=None, weight=p, bias=None, kind=1, rows=4, d=64, x_out=None, ldq=64):
        return handle.da_norm_int8(x, x_dtype, d, branch, 1, d, weight, 2, bias, 2, kind, rows, d, eps, x_out, d, p, ldq,
                                   p, None)

    assert norm(x=None) == _lib.DA_ERR_NULL
    assert norm(branch=p) == _lib.DA_ERR_NULL            # a branch needs x_out
    assert norm(kind=3) == _lib.DA_ERR_UNSUPPORTED
    assert norm(kind=0) == _lib.DA_ERR_UNSUPPORTED       # the quantiser takes no weight
    assert norm(bias=p) == _lib.DA_ERR_UNSUPPORTED       # nor an RMS norm a bias
    assert norm(rows=0) == _lib.DA_ERR_SHAPE
    assert norm(ldq=63) == _lib.DA_ERR_SHAPE
    assert norm(x_dtype=5) == _lib.DA_ERR_DTYPE

    def gemm(a=p, lda=64, ldb=64, bias=None, bias_dtype=2, ldc=32, c_dtype=1, m=8, n=32, k=64):
        return handle.da_gemm_i8(a, lda, p, p, ldb, p, bias, bias_dtype, 0, p, ldc, c_dtype, m, n, k, p, None)

    assert gemm(a=None) == _lib.DA_ERR_NULL
    assert gemm(k=131072, lda=131072, ldb=131072) == _lib.DA_ERR_SHAPE   # the int32 sum could overflow
    assert gemm(lda=48) == _lib.DA_ERR_SHAPE
    assert gemm(ldc=31) == _lib.DA_ERR_SHAPE
    assert gemm(c_dtype=3) == _lib.DA_ERR_DTYPE
    assert gemm(bias=p, bias_dtype=9) == _lib.DA_ERR_DTYPE
    assert gemm(a=p + 4) == _lib.DA_ERR_ALIGN
    assert gemm(lda=72) == _lib.DA_ERR_ALIGN

    assert handle.da_checkpoint8(p, 2, 64, 4, 64, 0, None, 0, p, p, None) == _lib.DA_ERR_DTYPE
    assert handle.da_checkpoint8(p, 1, 64, 4, 64, 1, None, 64, p, p, None) == _lib.DA_ERR_NULL
    assert handle.da_checkpoint8(p, 1, 64, 0, 64, 0, None, 0, p, p, None) == _lib.DA_ERR_SHAPE
    assert handle.da_checkpoint8(p, 1, 64, 4, 64, 0, None, 0, p + 8, p, None) == _lib.DA_ERR_ALIGN
    assert handle.da_checkpoint8_restore(p, p, 4, 64, p, 7, 64, None) == _lib.DA_ERR_DTYPE
    assert handle.da_checkpoint8_gelu_bwd(p, 1, 64, p, p, 4, 64, p, 63, None, 0, None) == _lib.DA_ERR_SHAPE
    assert handle.da_checkpoint8_wgrad_workspace_elems(0, 8, 8) == -1
    elems = handle.da_checkpoint8_wgrad_workspace_elems(64, 8, 8)
    assert elems >= 0

    def wgrad(dy=p, ldy=8, out_dtype=2, ldo=8, work=p, n=elems):
        return handle.da_checkpoint8_wgrad(dy, 1, ldy, p, p, 64, 8, 8, p, out_dtype, ldo, work, n, p, None)

    assert wgrad(dy=None) == _lib.DA_ERR_NULL
    assert wgrad(out_dtype=0) == _lib.DA_ERR_DTYPE       # neither fp32 nor dy's dtype
    assert wgrad(ldo=7) == _lib.DA_ERR_SHAPE
    assert wgrad(ldy=12) == _lib.DA_ERR_ALIGN
    if elems:
        assert wgrad(n=elems - 1) == _lib.DA_ERR_WORKSPACE


def test_eight_bit_operators_refuse_cpu_tensors() -> None:
    import torch
    import torch.nn as nn

    import double_attention_b200 as da

    x, q = torch.zeros(2, 32), torch.zeros(2, 32, dtype=torch.int8)
    with pytest.raises(ValueError):
        da.quantize_int8(x)
    with pytest.raises(ValueError):
        da.add_rmsnorm_int8(x, x, nn.RMSNorm(32).requires_grad_(False))
    with pytest.raises(ValueError):
        da.int8_linear(da.Int8Rows(q, torch.zeros(2)), da.Int8Rows(q, torch.zeros(2)))
    with pytest.raises(ValueError):
        da.checkpoint8(x.bfloat16())
    with pytest.raises(NotImplementedError):
        da.linear_checkpoint8(torch.zeros(2, 128), nn.Linear(128, 128))
