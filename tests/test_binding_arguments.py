"""What the binding takes for an ``int32_t`` argument: everything that ``ctypes.c_int32`` does."""
import ctypes

import numpy as np
import pytest

import cleave_b200 as cb


class Carrier:
    def __init__(self, value):
        self._as_parameter_ = value


class Whole:
    def __index__(self):
        return 40


@pytest.mark.parametrize("forty", [40, np.int64(40), np.uint8(40), Whole(), ctypes.c_int32(40), Carrier(ctypes.c_int32(40)), Carrier(40)])
def test_integers_and_c_integers_are_taken(forty):
    assert cb.lib().cleave_cuda_e4m3_bytes(3, forty) == 3 * 48
    assert cb.lib().cleave_cuda_e4m3_bytes(forty, 3) == 40 * 16


def test_truth_values_are_integers():
    assert cb.lib().cleave_cuda_e4m3_bytes(True, 3) == 16


@pytest.mark.parametrize("bad", [40.0, "40", None, np.float32(40), ctypes.c_float(40), Carrier("40")])
def test_the_rest_is_refused(bad):
    with pytest.raises(ctypes.ArgumentError):
        cb.lib().cleave_cuda_e4m3_bytes(3, bad)
