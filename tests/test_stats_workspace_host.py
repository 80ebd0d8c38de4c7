"""The room that head_stats asks for, as its documentation states it: bytes a position, by the vocabulary and the number of tokens
wanted."""
import pytest

N = 4096                                   # a multiple of the 256 rows that the room is counted in; the rest is a few hundred bytes


@pytest.mark.parametrize('V,d,top,notes', [
    (50304, 768, 0, 0), (50304, 768, 5, 1 / 8), (40000, 64, 32, 1 / 8), (32768, 768, 8, 1 / 4), (5003, 200, 20, 1 / 4), (2048, 768, 14, 1 / 4),
    (2048, 768, 32, 4), (1265, 608, 20, 4), (1265, 608, 8, 1 / 4), (256, 64, 8, 4), (256, 64, 1, 1 / 4), (2049, 768, 32, 1 / 4)])
def test_bytes_a_position(V, d, top, notes):
    from asrn_b200 import _lib
    assert (notes == 4) == (0 < top and V <= 2048 and V * V <= 24 * top * top * d)
    each = _lib.lib().asrn_head_stats_workspace_bytes(N, V, d, top, 0) / N
    want = (1 / 4 + notes) * V
    assert want <= each <= want + 64 + 128 + 16          # whole tiles of 256 columns, whole chunks of 32 scores, a position's own
