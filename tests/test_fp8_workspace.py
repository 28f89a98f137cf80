"""The workspace of the e4m3 product where the general kernel runs, which takes none (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest

from slipstream_amd import _ffi


@pytest.mark.parametrize("m,n,k", [(3, 130, (1 << 21) + 16), (3, 130, (1 << 21) + 1), (1 << 31, 8, 128), (8, 1 << 31, 128)])
@pytest.mark.parametrize("whole", [0, 1])
def test_no_copies_are_asked_for_that_no_kernel_reads(m, n, k, whole):
    """Rows beyond the reach of the DMA kernels' descriptors, and more of them than these count: both operands' copies
    were asked for (a second weight)."""
    need = ctypes.c_int64(-1)
    assert _ffi.lib().ss_fp8_workspace_size(m, n, k, whole, whole, _ffi.SS_DTYPE_BF16, ctypes.byref(need)) == _ffi.SS_OK
    assert need.value == 0
