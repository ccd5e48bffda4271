"""The C entry of the experts' product where tokens have no choices, on the CPU (no kernel is launched)."""
from __future__ import annotations

import ctypes

from practice_cuda_amd import _lib

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced


def test_tokens_without_choices_have_no_rows():
    L = _lib.lib()

    def call(a_rows, pairs, choices, order=None, b=FAKE):
        return L.pcamd_expert_bmm_int8(FAKE, a_rows, b, 3, 8, 32, 32, 256, 32, FAKE, _lib.BF16, 8, None, 0, 0, 0,
                                       FAKE, 1, FAKE, 8, 1, FAKE, order, pairs, choices, 0, None)

    assert call(3, 0, 0) == _lib.OK and call(3, 0, 0, order=FAKE) == _lib.OK and call(0, 0, 0) == _lib.OK
    assert call(3, 0, 1) == _lib.ERR_INVALID and call(3, 0, 1, order=FAKE) == _lib.ERR_INVALID
    assert call(3, 6, 0, order=FAKE) == _lib.ERR_INVALID
