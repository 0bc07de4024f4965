"""The mark of a tensor with scales of any value, on the host side."""
import pytest

import cleave_b200 as cb

ANY = 16


@pytest.mark.parametrize("rows,cols", [(1, 1), (200, 1000), (2 ** 31 - 1, 130)])
def test_a_marked_form_has_as_many_scales(rows, cols):
    L = cb.lib()
    for blocks in (1, 2, 3):
        assert L.cleave_cuda_e4m3_scales(rows, cols, blocks | ANY) == L.cleave_cuda_e4m3_scales(rows, cols, blocks) > 0
    for blocks in (0, 4, 32, 33):
        assert L.cleave_cuda_e4m3_scales(rows, cols, blocks | ANY) == 0
