"""How large the paged cache's tables may be; no GPU."""

import ctypes

import pytest


def test_pages_of_all_sequences_are_counted_in_32_bits():
    """Rows of cu that rise and fall could have every sequence ask for a whole row of the table."""
    from leankv_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(16)
    for seqs, width in ((2048, 1 << 20), (2048, (1 << 20) - 1), (65, 1 << 25), (31, 1 << 25)):
        st = ctypes.byref(_lib.PagesStruct(16, 16, 16, 16, 16, 1, 8, 1, 16, seqs, width, _lib.LKV_DTYPE_F16))
        assert lib.lkv_pages_extend(st, None, p, 0, None) == -1  # (without a workspace: nothing is launched)
        assert ("2^31" if seqs * (width + 1) >= 2 ** 31 else "workspace") in _lib.last_error()


def test_constructor_refuses_tables_past_that():
    from leankv_amd.paged import PagedKV

    with pytest.raises(ValueError, match="too large"):
        PagedKV(1, 1, 8, 2048, 1 << 24, page_size=16)
