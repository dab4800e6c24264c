"""Arguments of the 4-bit calls that are refused before any call, without a GPU."""
import numpy as np
import pytest
import torch


def test_slots_past_64_bits_are_refused():
    """An unsigned slot of 2^63 and more would turn into a negative one, whose row is skipped."""
    from pion_b200 import _lib, fp4
    for bad in ([2 ** 63], np.array([1, 2 ** 64 - 1], np.uint64)):
        with pytest.raises(ValueError):
            fp4._slots(None, bad, _lib.MEM_HOST)
    good = fp4._slots(None, np.array([1, 2 ** 63 - 1], np.uint64), _lib.MEM_HOST)
    assert good.tolist() == [1, 2 ** 63 - 1]
    assert fp4._slots(None, np.zeros(0, np.uint64), _lib.MEM_HOST).numel() == 0
