"""CPU: how grouped-query attention divides its calls, as the workspace sizes of
its host code tell it (no device work)."""

import pytest


@pytest.fixture(scope="module")
def size():
    from ernie_kv import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libernie_kv.so not built (run __graft_entry__.build())")
    return _lib.load().ekv_gqa_attention_workspace_size


@pytest.mark.parametrize("dim,group", [(64, 8), (128, 8), (256, 12)])
@pytest.mark.parametrize("seqs,kv", [(1, 1), (1, 8), (2, 8), (4, 8)])
def test_parts_of_many_rows_grow_with_the_pages(size, dim, group, seqs, kv):
    """One more page never makes the parts of a call fewer and longer while all
    of them run at once, one to a CU, and a row has up to 64."""
    rows = 128 // group  # one tile
    most = 4 * min(256 // (seqs * kv), 64)
    sizes = [size(seqs * rows, seqs, rows, 64 * pages, kv * group, kv, dim, 0) for pages in range(9, most + 1)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0


def test_a_second_kernel_only_where_it_may_find_rows(size):
    """Single rows beside chunks at long bounds take the kernel of few rows, in
    parts; chunks alone, and calls of short bounds, are one launch without parts."""
    assert size(513, 2, 512, 131072, 64, 8, 128, 0) > 0
    assert size(2051, 7, 512, 131072, 64, 8, 128, 0) > 0
    assert size(1024, 2, 512, 131072, 64, 8, 128, 0) == 0
    assert size(513, 2, 512, 8000, 64, 8, 128, 0) == 0
    assert size(513, 2, 512, 131072, 64, 8, 128, 1000) == 0
