"""Which tiles the paged attention takes, as its workspace shows: the host alone decides."""
import pytest

from qtpytorch_amd import _lib as L


def _rows(q_type, rows, D, B=16, G=4):
    """Rows of a tile for B sequences with `rows` rows a key head each, contexts of 4096 positions."""
    T = B * rows // G
    assert T * G == B * rows
    nbytes = L.lib().mxk_kv_pages_attend_workspace(q_type, T, B, 128, 32, 8, 8 * G, D)
    # a share of the line: two parts of a tile, what tile they are of, and for large tiles a word of bits
    fits = [r for r in (16, 128, 256) if nbytes % (2 * r * (4 * D + 8) + 32 + (4 if r > 16 else 0)) == 0]
    assert nbytes and len(fits) == 1
    return fits[0]


@pytest.mark.parametrize("q_type,D,last_small,last_middle", [
    (L.MXK_IN_BF16, 64, 64, 128), (L.MXK_IN_BF16, 128, 64, 128), (L.MXK_IN_F16, 128, 64, 128), (L.MXK_IN_BF16, 256, 96, None),
    (L.MXK_IN_F16, 256, 96, None), (L.MXK_IN_F32, 64, 96, None), (L.MXK_IN_F32, 128, 96, None), (L.MXK_IN_F32, 256, 96, None)])
def test_rows_of_a_tile(q_type, D, last_small, last_middle):
    assert _rows(q_type, 4, D) == _rows(q_type, last_small, D) == 16
    assert _rows(q_type, last_small + 4, D) == 128
    assert _rows(q_type, last_middle or 2000, D) == 128
    if last_middle:
        assert _rows(q_type, last_middle + 4, D) == 256
