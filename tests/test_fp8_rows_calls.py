"""Calls of the 8-bit row functions (vectors_b200/fp8.py, include/vx.h) that their documentation allows and
that are easily got wrong: calls with nothing to do, all operand types in every form, repeated and
concurrent small calls.  The definition and the tolerances are those of test_fp8_rows.py.
"""
import numpy as np
import pytest

import vectors_b200 as vx
import vectors_b200._native as N
from tests.test_fp8_rows import _bytes, _dtype, _grouped_want, _store, bound, decode, encode, rows_of


@pytest.mark.gpu
@pytest.mark.parametrize("max_rows", [5, 0])
def test_no_groups_and_no_offsets(max_rows):
    """No groups need no offsets, and leave the results as they are (which have a column for every stored
    row here, more than max_rows)."""
    import torch

    codes, scales = vx.fp8_empty(40, 100)
    q = torch.randn(3, 100, device="cuda")
    out = torch.full((3, 40), -7.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for offsets in (None, torch.zeros(1, dtype=torch.int64, device="cuda").data_ptr()):
        status = N.lib().vx_fp8_scores_grouped_device(0, q.data_ptr(), N.VX_F32, None, 3, 100, offsets, codes.data_ptr(),
                                                      scales.data_ptr(), 40, offsets, 0, 100, out.data_ptr(), N.VX_F32, 40,
                                                      max_rows, stream)
        assert status == 0, N.last_error()
    vx.fp8_check()
    assert (out == -7).all()
