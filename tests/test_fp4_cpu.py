"""Microscaled 4-bit rows without a GPU: store sizes, refusals, and the float64 definition the
GPU tests compare with against hand-derived values."""
import ctypes

import numpy as np
import pytest

import fp4_plain as plain


def test_sizes_and_refusals():
    from pion_b200 import _lib
    lib = _lib.load()
    c, s = ctypes.c_int64(), ctypes.c_int64()

    def sizes(fmt, n, dim):
        rc = lib.pion_v_b200_fp4_sizes(fmt, n, dim, ctypes.byref(c), ctypes.byref(s))
        return rc, c.value, s.value

    assert sizes(_lib.FP4_MX, 1000, 1536) == (0, 768000, 8 * 12 * 512)
    assert sizes(_lib.FP4_NV, 1000, 1536) == (0, 768000, 8 * 24 * 512)
    assert sizes(_lib.FP4_NV, 129, 100) == (0, 129 * 64, 2 * 2 * 512)
    assert sizes(_lib.FP4_MX, 0, 1) == (0, 0, 0)
    assert sizes(_lib.FP4_NV, 100000000, 1536)[1:] == (76800000000, 781250 * 24 * 512)
    assert sizes(2, 10, 10)[0] == _lib.EINVAL
    assert sizes(0, -1, 10)[0] == _lib.EINVAL
    assert sizes(0, 10, 0)[0] == _lib.ESHAPE
    assert sizes(0, 10, 8193)[0] == _lib.ESHAPE
    assert sizes(0, 1 << 31, 64)[0] == _lib.ESHAPE
    assert lib.pion_v_b200_fp4_sizes(0, 1, 1, None, None) == _lib.EINVAL


def test_workspace_and_null_contexts():
    from pion_b200 import _lib
    lib = _lib.load()
    d = _lib.FP4RowsDesc(_lib.FP4_NV, 0, 100000, 1536, 256, 256, 256, 256, 256)
    ws = lambda n, nq, k: lib.pion_v_b200_fp4_workspace(ctypes.byref(d), n, nq, k)  # noqa: E731
    assert ws(100000, 0, 10) == 0 and ws(0, 5, 10) == 0
    assert 0 < ws(100000, 1, 0) < ws(100000, 1, 10) < ws(100000, 4096, 10)
    assert ws(100000, 1 << 20, 10) == ws(100000, 4096, 10)     # searched in chunks
    assert ws(100001, 1, 10) == _lib.ESHAPE and ws(100, 1, 257) == _lib.ESHAPE
    assert ws(-1, 1, 1) == _lib.EINVAL and ws(1, -1, 1) == _lib.EINVAL
    assert lib.pion_v_b200_fp4_workspace(None, 1, 1, 1) == _lib.EINVAL
    assert lib.pion_v_b200_ctx_device(None) == _lib.EINVAL
    assert lib.pion_v_b200_fp4_clear(None, ctypes.byref(d), None) == _lib.EINVAL
    assert lib.pion_v_b200_fp4_write(None, ctypes.byref(d), None, 0, 0, 0, None, 0, 1,
                                     None) == _lib.EINVAL
    assert lib.pion_v_b200_fp4_read(None, ctypes.byref(d), None, 0, 0, None, 0, 0, 1,
                                    None) == _lib.EINVAL
    assert lib.pion_v_b200_fp4_scores(None, ctypes.byref(d), 1, None, 0, 0, 0, None, 0, 0, None, 0,
                                      1, None) == _lib.EINVAL
    assert lib.pion_v_b200_flat_fp4_knn(None, ctypes.byref(d), 1, 0, None, 0, 0, 0, 1, None, None,
                                        None, 0, 1, None) == _lib.EINVAL


def test_store_arguments():
    import torch

    import pion_b200
    with pytest.raises(ValueError):
        pion_b200.FP4Rows(4, 16, "e5m2")
    with pytest.raises(pion_b200.PionError):
        pion_b200.FP4Rows(4, 0)
    with pytest.raises(ValueError):
        pion_b200.FP4Rows(4, 16, "nv", codes=torch.zeros((4, 64), dtype=torch.uint8))
    with pytest.raises(ValueError):  # host tensors
        pion_b200.FP4Rows(4, 16, "nv", codes=torch.zeros((4, 64), dtype=torch.uint8),
                          scales=torch.zeros(2 * 512, dtype=torch.uint8),
                          row_scale=torch.zeros(4), norm_max=torch.zeros(1))


def test_desc_mirrors_the_header():
    from pion_b200 import _lib
    f = _lib.FP4RowsDesc
    offs = [f.format.offset, f.n_rows.offset, f.dim.offset, f.codes.offset, f.scales.offset,
            f.row_scale.offset, f.norm_max.offset, f.claim.offset]
    assert offs == [0, 8, 16, 24, 32, 40, 48, 56] and ctypes.sizeof(f) == 64


def test_definition_known_answers():
    # MX: a block whose largest magnitude is 5 has s = 2^(2 - 2) = 1
    x = np.zeros((1, 32))
    x[0, :9] = [5.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5.0, -0.2]
    codes, bits, g = plain.quantise(x, "mx")
    assert bits[0, 0] == 127 and g[0] == 1.0
    # 5 is halfway between 4 (code 6) and 6 (code 7): the even code; so are the others
    assert codes[0, :9].tolist() == [6, 0, 2, 2, 4, 4, 6, 14, 8]
    assert plain.values(codes, bits, "mx")[0, :8].tolist() == [4, 0, 1, 1, 2, 2, 4, -4]
    # NV: amax 2688 gives g = 1, its block s = 448, and codes on the grid of 448
    x = np.zeros((1, 32))
    x[0, 0], x[0, 1], x[0, 16] = 2688.0, -1344.0, 6.0
    codes, bits, g = plain.quantise(x, "nv")
    assert g[0] == 1.0 and plain.E4M3[bits[0, :2]].tolist() == [448.0, 1.0]
    assert codes[0, [0, 1, 16]].tolist() == [7, 8 + 5, 7]
    # saturation of the power-of-two scale: 7.9 lies past 6 s
    codes, bits, _ = plain.quantise(np.array([[7.9]]), "mx")
    assert plain.values(codes, bits, "mx")[0, 0] == 6.0


def test_layout_round_trip():
    rng = np.random.default_rng(0)
    bits = rng.integers(0, 256, (300, 24)).astype(np.uint8)
    flat = plain.store_scales(bits, 300)
    assert np.array_equal(plain.row_scales(flat, 300, 6), bits)
    r, b = 177, 13
    assert flat[((1 * 6 + 3) * 32 + r % 32) * 16 + (r % 128) // 32 * 4 + 1] == bits[r, b]


def test_slots_and_shapes_are_refused_before_any_call():
    import pion_b200
    import torch
    from pion_b200 import _lib, fp4
    assert fp4._slots(None, [3, -1], _lib.MEM_HOST).tolist() == [3, -1]
    assert fp4._slots(None, np.array([3, 1], np.uint8), _lib.MEM_HOST).dtype == torch.int64
    assert fp4._slots(None, [], _lib.MEM_HOST).numel() == 0
    for bad in ([1.5], [True], np.array([1.0, 2.0]), [[1]]):
        with pytest.raises(TypeError):
            fp4._slots(None, bad, _lib.MEM_HOST)
    with pytest.raises(ValueError):
        pion_b200.quantize_rows_fp4(None, np.zeros(8, np.float32))
