"""Microscaled 4-bit numbers and draws from logits, without a GPU: the layout's description, and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

import mx4_plain as plain

SOME = 0x10000                                # an address that no refused call looks at


@pytest.fixture(scope="module")
def lib(spg):
    return spg.lib()


def _matrix(spg, rows=4, cols=64, codes=SOME, scales=SOME, pitch=None):
    return spg.abi.Mx4(codes, scales, rows, cols, -(-cols // 32) * 16 if pitch is None else pitch)


def test_layout(spg, lib):
    for cols in (1, 31, 32, 33, 128, 129, 777, 8192):
        assert lib.spgk_mx4_pitch(cols) == -(-cols // 32) * 16
        for rows in (1, 31, 128, 129, 1000):
            assert lib.spgk_mx4_scales_bytes(rows, cols) == -(-rows // 128) * -(-cols // 128) * 512
            r, b = np.meshgrid(np.arange(rows), np.arange(-(-cols // 32)), indexing="ij")
            places = plain.scale_place(cols, r, b)
            assert len(np.unique(places)) == places.size and places.max() < lib.spgk_mx4_scales_bytes(rows, cols)
            for row, block in ((0, 0), (rows - 1, 0), (rows // 2, -(-cols // 32) - 1)):
                assert lib.spgk_mx4_scale_index(cols, row, block) == plain.scale_place(cols, row, block)
    assert lib.spgk_mx4_scales_bytes(0, 5) == 0


def test_plain_form_of_the_rounding():
    """The oracle itself: every value between two neighbours goes to the nearer one, half way to the even code."""
    x = np.zeros((1, 32), np.float32)
    x[0, :16] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, 4.0, -0.25, -0.75, -5.0, 0.26, 0.74, 1e-30, -0.0]
    code, scale = plain.quantize(x)
    assert scale[0, 0] == 127
    assert list(plain.values(code, scale, 32)[0, :16]) == [0, 1, 1, 2, 2, 4, 4, 6, 4, 0, -1, -4, 0.5, 0.5, 0, 0]


@pytest.mark.parametrize("change", [dict(cols=0), dict(codes=0), dict(scales=0), dict(codes=SOME + 8), dict(scales=SOME + 4), dict(pitch=24), dict(pitch=16), dict(cols=0x7fffff01, pitch=0x40000000),
                                    dict(rows=0x7fffff01), dict(rows=0x7ffff000, cols=0x7ffff000, pitch=0x40000000)])
def test_bad_matrices_are_refused(spg, lib, change):
    good, bad = _matrix(spg), _matrix(spg, **change)
    assert lib.spgk_mx4_quantize(SOME, 2, 64, C.byref(bad), None) == -2
    assert b"spgk_mx4_quantize" in lib.spgk_error_string()
    assert lib.spgk_mx4_dequantize(C.byref(bad), SOME, 2, 64, None) == -2
    assert lib.spgk_layer_mx4(C.byref(bad), None, 6, C.byref(good), SOME, 2, 64, None, SOME, None) == -2
    assert lib.spgk_layer_mx4(C.byref(good), None, 6, C.byref(bad), SOME, 2, 64, None, SOME, None) == -2
    assert lib.spgk_layer_mx4(C.byref(good), None, 6, C.byref(good), SOME, 2, 64, C.byref(bad), SOME, None) == -2


def test_bad_rows_are_refused(spg, lib):
    m = C.byref(_matrix(spg))
    for x, kind, ld in ((SOME, 3, 64), (SOME, -1, 64), (0, 2, 64), (SOME + 2, 2, 64), (SOME + 1, 0, 64), (SOME, 2, 63)):
        assert lib.spgk_mx4_quantize(x, kind, ld, m, None) == -2, (x, kind, ld)
        assert lib.spgk_mx4_dequantize(m, x, kind, ld, None) == -2, (x, kind, ld)
    assert lib.spgk_mx4_quantize(SOME, 2, 64, None, None) == -2
    none = C.byref(_matrix(spg, rows=0, codes=0, scales=0))
    assert lib.spgk_mx4_quantize(0, 2, 64, none, None) == 0 and lib.spgk_mx4_dequantize(none, 0, 2, 64, None) == 0


def test_bad_layers_are_refused(spg, lib):
    w, x, other = _matrix(spg, rows=48), _matrix(spg), _matrix(spg, cols=96)
    nxt, wrong = _matrix(spg, cols=48), _matrix(spg, rows=5, cols=48)

    def call(w=w, bias=0, act=6, x=x, y=SOME, kind=2, ldy=48, nxt=None, status=SOME):
        return lib.spgk_layer_mx4(C.byref(w), bias, act, C.byref(x), y, kind, ldy, None if nxt is None else C.byref(nxt), status, None)
    assert call(x=other) == -2 and call(w=_matrix(spg, rows=0)) == -2
    assert call(act=7) == -2 and call(act=-1) == -2 and call(y=0) == -2 and call(kind=3) == -2 and call(y=SOME + 2) == -2 and call(y=SOME + 1, kind=0) == -2
    assert call(ldy=47) == -2 and call(status=0) == -2 and call(bias=SOME + 2) == -2
    wide = _matrix(spg, cols=(1 << 27) + 32)
    assert call(w=wide, x=wide, ldy=4) == -2
    assert call(nxt=wrong) == -2 and call(nxt=other) == -2 and call(nxt=nxt, act=5) == -2
    assert call(x=_matrix(spg, rows=0)) == 0


def test_bad_draws_are_refused(lib):
    def call(logits=SOME, kind=2, ld=10, n=2, width=10, u=SOME, tokens=SOME, temperature=0, probs=0):
        return lib.spgk_sample_rows(logits, kind, ld, n, width, temperature, 0, 0, 0, u, tokens, probs, 0, None)
    for bad in (dict(kind=3), dict(width=0), dict(width=262145, ld=262145), dict(logits=0), dict(u=0), dict(tokens=0), dict(logits=SOME + 2), dict(ld=9), dict(temperature=SOME + 2), dict(probs=SOME + 1)):
        assert call(**bad) == -2, bad
        assert b"spgk_sample_rows" in lib.spgk_error_string()
    assert call(n=0) == 0
