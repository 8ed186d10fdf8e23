"""Tables of a packed batch put together by hand: sizes that do not fit are refused on the host (the kernels read as many entries as the sizes say)."""
import pytest
import torch

from tensoflow_amd import ops

z = lambda n, t=torch.int64: torch.zeros(n, dtype=t)


@pytest.mark.parametrize("n_rows,n_segments,offsets,index,starts,name", [
    (70, 2, z(2), z(70), z(2), "offsets"), (70, 2, z(3), z(69), z(2), "index"), (70, 2, z(3), None, z(1), "starts"), (70, 2, z(3), z(70), None, "starts"),
    (70, 2, None, z(70), z(2), "offsets"), (70, 2, z(3, torch.int32), z(70), z(2), "offsets"), (70, 2, z(3), z(70, torch.int32), z(2), "index"),
    (70, 2, z(3), z(140)[::2], z(2), "index"), (64, 0, z(0), None, z(1), "offsets"), (65, 1, z(2), None, z(1), "starts")])
def test_tables_that_do_not_fit(n_rows, n_segments, offsets, index, starts, name):
    with pytest.raises(RuntimeError, match=name):
        ops.SegmentTables(n_rows, n_segments, offsets, index, None, starts)


def test_tables_that_fit():
    t = ops.SegmentTables(70, 2, z(3), z(70), None, z(2))
    assert (t.n_rows, t.n_segments, t.position, t.block_table, t.slots) == (70, 2, None, None, None)
    assert ops.SegmentTables(0, 0, z(1), None, None, z(0)).index is None
