"""How many tokens a sequence's page table may hold in the decode kernels, on the
CPU: token numbers are 32 bits wide and run ahead of the last token by the tiles
that are on their way."""
from __future__ import annotations

import ctypes

import pytest

from practice_cuda_amd import _lib

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first


def decode(page, max_pages):
    """A call without the workspace that it needs: it is refused in any case."""
    L = _lib.lib()
    rc = L.pcamd_latent_decode(FAKE, FAKE, _lib.BF16, 1, 1, 16, 512, 64, 8192, 8192, 512, 1024, 1024, 64, FAKE,
                               _lib.BF16, 0, 0, FAKE, 0, 0, None, 0, 0, 1, page, FAKE, max_pages, max_pages, FAKE,
                               FAKE, 8192, 8192, 512, None, 0, 0, 0, 0.1, None, 0, None)
    return rc, L.pcamd_last_error()


@pytest.mark.parametrize("page,max_pages", [(2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (2 ** 30, 2), (2 ** 31 - 600, 1),
                                            (2 ** 31 - 1023, 1), (1023, 2099202), (7, 306783378)])
def test_tables_that_end_near_2_31_tokens_are_refused(page, max_pages):
    L = _lib.lib()
    assert page * max_pages > 2 ** 31 - 1024
    assert L.pcamd_latent_decode_workspace(1, 1, 16, 512, page, max_pages) == _lib.ERR_UNSUPPORTED
    assert b"tokens a sequence" in L.pcamd_last_error()
    rc, error = decode(page, max_pages)
    assert rc == _lib.ERR_UNSUPPORTED and b"tokens a sequence" in error


@pytest.mark.parametrize("page,max_pages", [(2 ** 31 - 1024, 1), (1, 2 ** 31 - 1024), (2 ** 20, 2047), (64, 2 ** 25 - 16)])
def test_the_largest_tables_are_taken(page, max_pages):
    assert _lib.lib().pcamd_latent_decode_workspace(1, 1, 16, 512, page, max_pages) > 0
    rc, error = decode(page, max_pages)
    assert rc == _lib.ERR_INVALID and b"workspace" in error
