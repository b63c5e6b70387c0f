"""Sizes at the limits of the 8-bit cache's entry points, refused before a launch."""
import ctypes as C

import pytest

D = C.c_void_p(16)  # never dereferenced: every call below is refused


@pytest.fixture(scope="module")
def lib(tq4):
    return tq4.kv8._lib()


def test_rows_of_a_streamed_call_with_many_records(lib):
    """The join takes workgroups of 1024 for rows of more than 32 records, those of
    few sequences in shares among them: fewer than 2^22 rows then. (-6 is the missing
    workspace of a call within the bounds.)"""
    def pre(rows, max_blocks, B=2):
        return lib.tq4_kv8_paged_prefill(None, 1, 0, D, D, D, D, D, D, D, None, 0, D, 8 * 128,
                                         rows, B, 8, 1, 128, 16, 64, max_blocks, 4, 1, 0.1)
    assert pre(2 ** 19 - 1, 2 ** 16) == -6
    assert pre(2 ** 19, 2 ** 16) == pre(2 ** 20, 2 ** 16) == -10
    # 32 records and fewer: 2^24
    assert pre(2 ** 21 - 1, 2 ** 16, B=16) == -6
    assert pre(2 ** 21, 2 ** 16, B=16) == -10
