"""The longest rows that the int8 quantizer takes, on the CPU (no kernel is launched on these paths)."""
from __future__ import annotations

import ctypes

import pytest

from practice_cuda_amd import _lib

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first


@pytest.mark.parametrize("n", [2**31 - 16384, 2**31 - 8192, 2**31 - 17, 2**31 - 1])
def test_quant_entry_refuses_the_longest_rows(n):
    """A long row's threads step on by 1024 * 8 values, past the row's end by up to as many, which has to fit 32 bits."""
    L = _lib.lib()
    assert L.pcamd_quant_int8(FAKE, _lib.BF16, 1, 1, n, 0, n, FAKE, 0, 2**31, FAKE, 0, 1, 1e-12, None) == -2
    assert b"columns" in L.pcamd_last_error()
