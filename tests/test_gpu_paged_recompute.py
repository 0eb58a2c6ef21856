"""Which sequences of a chunk are computed again by the kernel for few tokens: those with rows that a masked value has spoilt.

The flags are read from the workspace that the call is given: 16 bytes of counts, then a 32-bit word a sequence.
"""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_paged import BF16, FP16, Case

from double_attention_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def _spoilt(case: Case, per_map: bool = False) -> list[int]:
    """Flags of the sequences of one call on the C entry point, given a workspace that this reads afterwards."""
    lib, batch = _lib.lib(), case.batch
    tokens, sequences, columns = case.q.shape[1], len(case.held), batch.table.shape[1]
    code = _lib.DA_BF16 if case.dtype == BF16 else _lib.DA_F16
    sizes = case.h, case.r, case.d, case.s
    need = lib.da_paged_attn_workspace_size(tokens, sequences, columns, case.page, batch.max_new, *sizes, int(per_map))
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    y = torch.empty(tokens, *((case.s,) if per_map else ()), case.d, dtype=case.dtype, device="cuda")
    weights = None if per_map or case.weights is None else case.weights.data_ptr()
    status = lib.da_paged_attn(
        case.q.data_ptr(), case.q.stride(0), case.q.stride(1), tokens, case.key_pages.data_ptr(), case.value_pages.data_ptr(), code,
        case.key_pages.shape[0], case.page, *sizes, batch.table.data_ptr(), batch.table.stride(0), columns,
        batch.lengths.data_ptr(), batch.starts.data_ptr(), sequences, batch.max_new, case.scales.data_ptr(), weights, int(per_map), 1,
        y.data_ptr(), work.data_ptr(), need, ops.workspace(y.device).status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert status == _lib.DA_OK
    flags = work[16:16 + 4 * sequences].view(torch.int32).tolist()
    assert ops.device_status() == 0
    return flags


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [16.0, 0.0, -16.0])
@pytest.mark.parametrize("shape", [(1, 1, 128, 256, 32), (2, 2, 128, 256, 64), (4, 4, 128, 512, 16), (1, 3, 64, 128, 64)])
@pytest.mark.parametrize("per_map", [False, True])
def test_numbers_leave_nothing_to_compute_again(shape, scale, dtype, per_map) -> None:
    case = Case(*shape, dtype, [100, 0, 700], [150, 17, 200], scale=scale, seed=21, fill=5.0)
    case.append()
    assert _spoilt(case, per_map) == [0, 0, 0]


def test_a_later_value_that_is_no_number_has_its_sequence_computed_again() -> None:
    case = Case(2, 2, 128, 256, 32, BF16, [100, 30], [200, 170], seed=22, fill=5.0)
    case.v[199, 7] = math.nan
    case.append()
    assert _spoilt(case) == [1, 0]


@pytest.mark.parametrize("sequences", [1, 2, 31, 32])
def test_chunks_alone_leave_the_other_kernel_the_rows_of_no_sequence(sequences) -> None:
    case = Case(1, 1, 64, 128, 16, BF16, [b % 5 for b in range(sequences)], [17 + b for b in range(sequences)], seed=23, behind=9)
    case.append()
    y = case.attend()
    case.check(y)
    assert not y[sum(case.new):].any()
