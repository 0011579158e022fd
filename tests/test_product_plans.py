"""How the head's product is cut, seen from the workspace that it asks for (no GPU needed: a B200's 148 multiprocessors are
assumed where there is no device)."""

import ctypes

import pytest

TILE = 256


def split_bytes(lib, rows, vocab, hidden):
    """What the workspace holds beside two states a row and column tile, and a value a row: the split tiles' sums."""
    n = ctypes.c_int64()
    assert lib.b2s_lmhead_logprobs_workspace(rows, vocab, hidden, ctypes.byref(n)) == 0
    tiles = -(-vocab // TILE)
    return n.value - -(-(rows * tiles * 32 + rows * 4) // 256) * 256


@pytest.mark.parametrize("rows,rest,hidden,split", [
    # faster whole: the merge costs more than the tile's way from HBM
    (16, 8, 1024, False), (128, 2, 1024, False), (16, 16, 1024, False), (16, 6, 2048, False), (128, 4, 2048, False),
    (16, 16, 4096, False), (128, 8, 4096, False),
    # faster split
    (1, 2, 4096, True), (16, 6, 4096, True), (128, 3, 4096, True), (16, 2, 2048, True), (16, 10, 8192, True)])
def test_left_over_column_tiles_are_split_where_that_is_faster(pkg, rows, rest, hidden, split):
    lib = pkg._native.capi()
    got = split_bytes(lib, rows, (2 * 148 + rest) * TILE, hidden)
    assert got == (8 * rest * rows * TILE * 4 if split else 0)
