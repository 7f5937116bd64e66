"""Sizes of the grouped operators that no launch holds (2^32 work-items in a dimension) are refused on the host."""
import ctypes

import numpy as np
import pytest

from hyperion_amd import _lib

P = ctypes.c_void_p(16)  # a pointer that is never followed: the call is refused before


def _refused(fn, *args):
    lib = _lib.load()
    assert getattr(lib, fn)(*args) == -1, fn
    return lib.hypmi_last_error().decode()


def test_more_work_than_a_launch_holds():
    def affine(n):
        return _refused("hypmi_grouped_affine", P, 0, 8, 8, P, P, 16, 1, n, n, None, P, P, None, 4, 0, P, 4, 4, None)

    for n in (1 << 23, (1 << 31) - 1):  # tiles of 512 work-items
        assert "too many workgroups" in affine(n)
    assert "too many groups" in _refused("hypmi_grouped_weights", P, P, 1 << 24, 4, 4, P, P, None)

    def score(kp, n):
        return _refused("hypmi_grouped_score", P, kp, P, kp, kp, P, P, P, P, 1, n, P, None)

    for kp, threads in ((8, 640), (152, 640), (192, 384), (512, 384)):
        for n in (-(-(1 << 32) // threads), 1 << 40):
            assert "too many workgroups" in score(kp, n)

    def gram(d, n):
        return _refused("hypmi_grouped_gram_f64", P, 0, d, d, None, P, P, P, 1, n, 0, None, P, P, None, 0, None)

    assert "too many" in gram(8, 1 << 24) and "too many" in gram(512, 1 << 20) and "too many" in gram(8, 1 << 60)
    # the second launch: a workgroup per group and pair of blocks
    assert "too many" in _refused("hypmi_grouped_gram_f64", P, 0, 512, 512, None, P, P, P, 1 << 17, 1 << 17, 1, None, P, P, P,
                                  1 << 40, None)
    assert "too many rows" in _refused("hypmi_q4_rows", P, 160, 150, P, P, 1, 1 << 24, P, P, P, None)
    for n in (1 << 24, 1 << 40):
        assert "too many workgroups" in _refused("hypmi_q4_score", P, P, P, 150, P, 152, P, P, P, P, P, 16, 256, 1, n, P, None)


def test_more_groups_than_the_search_for_a_group_counts():
    n = (1 << 30) + 1
    assert "bad shape" in _refused("hypmi_grouped_affine", P, 0, 8, 8, P, P, 16, n, 1, 1, None, P, P, None, 4, 0, P, 4, 4, None)
    assert "bad shape" in _refused("hypmi_grouped_pack", P, 8, 8, P, n, 1, P, P, P, None, 16, None)
    assert "bad shape" in _refused("hypmi_grouped_score", P, 40, P, 40, 40, P, P, P, P, n, 1, P, None)
    assert "bad shape" in _refused("hypmi_grouped_gram_f64", P, 0, 8, 8, None, P, P, P, n, n, 0, None, P, P, None, 0, None)
    assert "bad shape" in _refused("hypmi_q4_rows", P, 160, 150, P, P, n, 1, P, P, P, None)
    assert "bad shape" in _refused("hypmi_q4_score", P, P, P, 150, P, 152, P, P, P, P, P, 16, 256, n, 1, P, None)
    from hyperion_amd import engine

    with pytest.raises(ValueError, match="2.30 groups"):
        engine.RowGroups(np.zeros(n, np.int8))
