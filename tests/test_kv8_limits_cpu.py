"""Sizes at the limits of the 8-bit cache's entry points, refused before a launch."""
import ctypes as C

import pytest
import torch

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


def test_sizes_past_32_bits_are_not_cut(tq4):
    """Whole numbers that the C ABI's 32-bit sizes do not hold are refused, not taken
    modulo 2^32; a max_query_len of any size past the rows means the rows."""
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for block_size in (2 ** 32 + 16, 16 - 2 ** 32, -16):
        with pytest.raises(ValueError, match="block_size"):
            tq4.paged_plan(i(3), i(3), i(3, 4), i(9), i(2), i(5), i(4), i(3), block_size)
    dec = [2, 8, 2, 128, 16, 64, 4]
    for k in range(7):
        for n in (2 ** 32 + dec[k], dec[k] - 2 ** 32):
            with pytest.raises(ValueError, match="must lie in"):
                tq4.kv8_decode_workspace_bytes(*dec[:k], n, *dec[k + 1:])
    pre = [9, 2, 8, 2, 128, 16, 64]
    for k in range(7):
        for n in (2 ** 32 + pre[k], pre[k] - 2 ** 32):
            with pytest.raises(ValueError, match="must lie in"):
                tq4.kv8_prefill_workspace_bytes(*pre[:k], n, *pre[k + 1:], 4)
    with pytest.raises(ValueError, match="must lie in"):
        tq4.kv8_prefill_workspace_bytes(*pre, -4)
    # 200 rows of heads enough for row tiles: 4 of them a sequence need another size
    pre = [200, 2, 8, 2, 128, 16, 4000]
    whole = tq4.kv8_prefill_workspace_bytes(*pre, 200)
    assert whole != tq4.kv8_prefill_workspace_bytes(*pre, 4)
    assert whole == tq4.kv8_prefill_workspace_bytes(*pre, 2 ** 32 + 4)
