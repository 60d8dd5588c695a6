"""Workspaces of attention over pages: bounded where many sequences may be long; no GPU."""

import pytest


def _lib():
    from leankv_amd import _lib

    return _lib.load()


@pytest.mark.parametrize("heads,kv", [(32, 8), (8, 8), (32, 2), (64, 8), (40, 1), (16, 1)])
@pytest.mark.parametrize("max_len", [8192, 131072, 1 << 20, (1 << 30) - 256])
def test_decode_workspace_is_bounded(heads, kv, max_len):
    """256 MB, but for as many splits as two workgroups for each of 256 CUs need, and their rows."""
    for seqs in (1, 2, 8, 100, 256, 2048):
        need = _lib().lkv_pages_decode_attn_workspace_bytes(seqs, heads, kv, max_len)
        assert need <= max(1 << 28, 520 * (512 + seqs * kv) * (heads // kv)), (seqs, need)


def test_few_rows_workspace_is_bounded():
    for max_len in (131072, 1 << 20):
        for seqs, new in ((2048, 1), (256, 8), (8, 5)):
            need = _lib().lkv_pages_prefill_attn_workspace_bytes(seqs * new, seqs, 32, 8, new, max_len)
            assert need <= max(1 << 28, 520 * (512 + seqs * 8) * 4 * new), (seqs, need)


def test_two_sequences_have_records_of_two():
    """One head each, no group larger than there are sequences: three records a split."""
    need = _lib().lkv_pages_decode_attn_workspace_bytes(2, 2, 2, 65536)
    assert need == 2 * 2 * 128 * 3 * 520  # 512 workgroups for 4 pairs: 128 splits
