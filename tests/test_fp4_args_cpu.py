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


def test_a_lone_claim_buffer_is_refused():
    """A store is made of no given tensors, or of all but the claims: given alone, they would be
    dropped."""
    import pion_b200
    claim = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="claim"):
        pion_b200.FP4Rows(4, 16, "nv", device="cpu", claim=claim)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.float16])
def test_a_new_store_does_not_go_by_torchs_default_dtype(dtype):
    """A model's program often sets one: the kernels read and write float32 scales and norms."""
    import pion_b200
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        rows = pion_b200.FP4Rows(5, 16, "nv", device="cpu")
    finally:
        torch.set_default_dtype(before)
    assert rows.row_scale.dtype == rows.norm_max.dtype == torch.float32
    assert rows.codes.dtype == rows.scales.dtype == torch.uint8 and rows.claim.dtype == torch.int32
    assert torch.isnan(rows.row_scale).all() and rows.norm_max.item() == 0


def test_a_stores_tensors_and_sizes_stay():
    """The calls pass their addresses and sizes as they were at first: another tensor or size put in
    their place would not be seen, and the old memory freed."""
    import pion_b200
    rows = pion_b200.FP4Rows(5, 16, "nv", device="cpu")
    for name in ("codes", "scales", "row_scale", "norm_max", "claim", "n_rows", "dim", "format"):
        was = getattr(rows, name)
        with pytest.raises(AttributeError):
            setattr(rows, name, was)
        assert getattr(rows, name) is was



def test_numbers_past_64_bits_are_refused():
    """ctypes would wrap them: a start of 2^64 is not slot 0."""
    from pion_b200 import fp4
    for bad in (2 ** 64, 2 ** 63, -2 ** 63 - 1):
        with pytest.raises(ValueError):
            fp4._int64(bad, "start")
    for good in (0, -1, 2 ** 63 - 1, np.int64(7), np.uint32(9)):
        assert fp4._int64(good, "start") == good and type(fp4._int64(good, "start")) is int
    with pytest.raises(TypeError):
        fp4._int64(1.5, "start")
    import pion_b200
    with pytest.raises(ValueError):
        pion_b200.FP4Rows(2 ** 64 + 4, 16, "nv", device="cpu")
    with pytest.raises(ValueError):
        pion_b200.FP4Rows(4, 2 ** 64 + 16, "nv", device="cpu")
