"""What the table's gradient refuses for its size, before it has launched anything.  No device: a launch would fail with another status."""
import pytest

from pixienn_amd import capi

F32, BF16 = 0, 1
HERE = 64            # an address that no refused call reads


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("type,rows,width", [(BF16, (1 << 29) + 64, 1), (F32, (1 << 30) - 1, 7), (F32, (1 << 28) + 64, 257), (BF16, 1 << 20, 1 << 23)])
def test_more_than_a_grid_takes_is_refused_before_a_launch(accumulate, type, rows, width):
    # runs that go on from chunk to chunk are a workgroup for every 32 rows and 256 values
    args = (HERE, HERE, HERE, type, type, 0, rows, 8, width, width, width, 1.0, accumulate)
    assert capi.call_raw("pxh_embedding_backward", *args, HERE, 1 << 62, None) == -1
    assert "too many rows" in capi.last_error()
    # nor does it ask for memory first
    assert capi.call_raw("pxh_embedding_backward", *args, HERE, 0, None) == -1 and "too many rows" in capi.last_error()


def test_a_table_of_too_many_rows_is_refused_before_a_launch():
    # zeros are a workgroup for every 32 rows and 256 vectors
    args = (HERE, HERE, HERE, F32, F32, 0, 3, 1 << 30, 4096, 4096, 4096, 1.0, 0)
    assert capi.call_raw("pxh_embedding_backward", *args, HERE, 1 << 62, None) == -1 and "too many rows" in capi.last_error()
    # what is added to is not walked
    assert capi.call_raw("pxh_embedding_backward", *args[:-1], 1, HERE, 0, None) != 0 and "workspace too small" in capi.last_error()
