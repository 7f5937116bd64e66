"""Argument checks of the grouped operators and the 4-bit gallery that come before any device work."""
import ctypes

import numpy as np
import pytest

from hyperion_amd import _lib


def _refused(fn, *args):
    lib = _lib.load()
    assert getattr(lib, fn)(*args) == -1, fn
    return lib.hypmi_last_error().decode()


P = ctypes.c_void_p(16)  # a pointer that is never followed: the call is refused before


def test_sizes_are_checked_on_the_host():
    from hyperion_amd import engine

    for sizes, match in (([1, -1], "negative"), ([[1]], "1-D"), ([0.5], "integers")):
        with pytest.raises(ValueError, match=match):
            engine.RowGroups(sizes)
    with pytest.raises(ValueError, match="1-D"):
        engine.RowGroups.from_ids(np.zeros((2, 2), int))


def test_sizes_of_tables():
    lib = _lib.load()
    assert lib.hypmi_grouped_weights_bytes(3, 33, 17) == 3 * 2 * 2 * 2048
    assert lib.hypmi_grouped_columns_bytes(3, 17) == 3 * 2 * 32 * 4
    assert lib.hypmi_grouped_weights_bytes(3, 0, 17) == 0
    assert [lib.hypmi_grouped_score_rows(k) for k in (0, 7, 8, 192, 200, 512, 520)] == [0, 0, 128, 128, 64, 64, 0]
    assert lib.hypmi_grouped_gram_workspace_bytes(2, 33) == 2 * (3 * 1024 + 64) * 8
    assert lib.hypmi_grouped_gram_workspace_bytes(0, 33) == 0
    assert [lib.hypmi_q4_ksteps(k) for k in (0, 1, 150, 192, 193, 300, 512, 513)] == [0, 1, 5, 6, 8, 10, 16, 0]


def test_refusals_of_the_c_abi():
    def affine(x=P, kind=0, ldx=8, d=8, tile=64, w=P, m=4, y=P, ldy=4, n=1, cols=None):
        return _refused("hypmi_grouped_affine", x, kind, ldx, d, P, P, tile, n, 1, 1, None, w, P, None, m, 0, y, ldy, m if cols is None else cols, None)

    assert "null" in affine(x=None) and "null" in affine(w=None) and "null" in affine(y=None)
    assert "fp32, fp16 or bf16" in affine(kind=3) and "fp32, fp16 or bf16" in affine(kind=-1)
    assert "leading" in affine(ldx=7) and "leading" in affine(ldy=6, m=6) and "leading" in affine(ldy=4, m=5)
    assert "columns to write" in affine(cols=3) and "columns to write" in affine(m=2, cols=5, ldy=8)
    assert "16, 64 or 128" in affine(tile=48)
    assert "16-byte" in affine(y=ctypes.c_void_p(20))
    assert "bad shape" in affine(d=0) and "bad shape" in affine(n=-1)
    assert "null" in _refused("hypmi_grouped_weights", None, None, 1, 4, 4, P, P, None)
    assert "bad shape" in _refused("hypmi_grouped_weights", P, None, 1, 0, 4, P, P, None)

    def score(g1=P, ld=40, kp=40, s=P):
        return _refused("hypmi_grouped_score", g1, ld, P, ld, kp, P, P, P, P, 1, 1, s, None)

    assert "null" in score(g1=None) and "null" in score(s=None)
    assert "multiple of 8" in score(kp=36) and "multiple of 8" in score(kp=520, ld=520)
    assert "leading" in score(ld=32) and "leading" in score(ld=41)
    assert "16-byte" in score(g1=ctypes.c_void_p(8))

    def gram(x=P, kind=0, ldx=8, chunks=1, slots=0, ws=None, nbytes=0):
        return _refused("hypmi_grouped_gram_f64", x, kind, ldx, 8, None, P, P, P, 1, chunks, slots, None, P, None, ws,
                        nbytes, None)

    assert "fp32 or fp64" in gram(kind=1) and "leading" in gram(ldx=7) and "null" in gram()
    lib = _lib.load()
    assert lib.hypmi_grouped_gram_f64(P, 0, 8, 8, None, P, P, P, 1, 1, 2, None, P, P, P, 100, None) == -1
    assert b"workspace" in lib.hypmi_last_error()
    assert lib.hypmi_grouped_gram_f64(P, 0, 8, 8, None, P, P, P, 2, 1, 0, None, P, P, None, 0, None) == -1
    assert b"unit of work" in lib.hypmi_last_error()

    assert "coordinates" in _refused("hypmi_q4_rows", P, 600, 513, P, P, 1, 1, P, P, P, None)
    assert "bad shape" in _refused("hypmi_q4_rows", P, 30, 30, P, P, 1, 1, P, P, P, None)
    assert "null" in _refused("hypmi_q4_rows", P, 32, 30, P, P, 1, 1, None, P, P, None)

    def q4(codes=P, k=30, ld=32, tests=16, rows=64):
        return _refused("hypmi_q4_score", codes, P, P, k, P, ld, P, P, P, P, P, tests, rows, 1, 1, P, None)

    assert "null" in q4(codes=None) and "leading" in q4(ld=31) and "leading" in q4(ld=34) and "leading" in q4(k=33, ld=36)
    assert "multiple of 64" in q4(rows=96) and "multiple of 64" in q4(rows=0)
    assert "16, 32 or 64" in q4(tests=48) and "coordinates" in q4(k=0)
    assert "16-byte" in q4(codes=ctypes.c_void_p(8))

    def pack(s=P, ld=8, k=8, n=1, c=P, out=P, kp=16):
        return _refused("hypmi_grouped_pack", s, ld, k, P, 1, n, P, c, out, None, kp, None)

    assert "null" in pack(s=None) and "null" in pack(c=None) and "no result" in pack(out=None)
    assert "bad shape" in pack(ld=7) and "bad shape" in pack(kp=9) and "bad shape" in pack(k=0) and "bad shape" in pack(n=-1)


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.hypmi_grouped_affine(None, 0, 8, 8, None, None, 64, 0, 0, 0, None, None, None, None, 4, 0, None, 4, 4, None) == 0
    assert lib.hypmi_grouped_pack(None, 8, 8, None, 0, 0, None, None, P, None, 16, None) == 0
    assert lib.hypmi_grouped_score(None, 40, None, 40, 40, None, None, None, None, 0, 0, None, None) == 0
    assert lib.hypmi_grouped_gram_f64(None, 0, 8, 8, None, None, None, None, 0, 0, 0, None, None, None, None, 0, None) == 0
    assert lib.hypmi_q4_score(None, None, None, 30, None, 32, None, None, None, None, None, 16, 64, 0, 0, None, None) == 0
