"""8-bit numbers in blocks, layers on them and rows to experts and back, without a GPU: the layout's description, the plain forms themselves, and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain as plain

SOME = 0x10000                                # an address that no refused call looks at


@pytest.fixture(scope="module")
def lib(spg):
    return spg.lib()


def _matrix(spg, rows=4, cols=64, codes=SOME, scales=SOME, pitch=None):
    return spg.abi.Fp8(codes, scales, rows, cols, -(-cols // 16) * 16 if pitch is None else pitch)


def test_layout(spg, lib):
    for cols in (1, 15, 16, 17, 127, 128, 129, 511, 512, 513, 777, 8192):
        assert lib.spgk_fp8_pitch(cols) == -(-cols // 16) * 16
        for rows in (1, 31, 128, 129, 1000):
            assert lib.spgk_fp8_scales_bytes(rows, cols) == -(-plain.blocks(cols) // 4) * rows * 4
            r, b = np.meshgrid(np.arange(rows), np.arange(plain.blocks(cols)), indexing="ij")
            places = plain.scale_place(rows, r, b)
            assert len(np.unique(places)) == places.size and places.max() < lib.spgk_fp8_scales_bytes(rows, cols)
            for row, block in ((0, 0), (rows - 1, 0), (rows // 2, plain.blocks(cols) - 1)):
                assert lib.spgk_fp8_scale_index(rows, row, block) == plain.scale_place(rows, row, block)
    assert lib.spgk_fp8_scales_bytes(0, 5) == 0
    assert lib.spgk_fp8_scales_bytes(0x7fffff00, 0x7fffff00) == 0x400000 * 0x7fffff00 * 4      # beyond 32 bits


def test_plain_form_of_the_rounding():
    """The oracle itself: every value between two neighbours goes to the nearer one, half way to the even code; 448 is the largest in every block."""
    x = np.zeros((1, 128), np.float32)
    x[0, :14] = [448, 17, 19, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 440, 464 / 2, -17, -0.0, 1e-30, 2.0 ** -10 * 1.001]
    code, scale = plain.quantize(x)
    assert scale[0, 0] == 127
    got = plain.values(code, scale)[0, :14]
    for v, g in zip(x[0, :14].astype(float), got):
        gaps = np.abs(plain.SIZES[:127] - abs(v))
        assert abs(abs(v) - abs(g)) == gaps.min()
    for v, e in ((448.0, 127), (448.001, 128), (449 * 2.0 ** 20, 148), (1.75, 119), (1.7501, 120), (2.0 ** -126, 0), (2.0 ** -149, 0), (3.4e38, 247), (0.0, 0)):
        x[:] = 0
        x[0, 5] = v
        assert plain.quantize(x)[1][0, 0] == e, v


def test_plain_form_of_the_route():
    l = np.array([[1, 3, 3, 2], [-np.inf, np.nan, 0, -np.inf], [-np.inf] * 4, [np.inf, 5, np.inf, np.inf]])
    chosen, gates, starts, order, places = plain.route(l, 2, True)
    assert chosen.tolist() == [[1, 2], [2, -1], [-1, -1], [0, 2]]
    assert np.allclose(gates, [[0.5, 0.5], [1, 0], [0, 0], [0.5, 0.5]])
    assert starts.tolist() == [0, 1, 2, 5, 5] and order.tolist() == [3, 0, 0, 1, 3, -1, -1, -1] and places.tolist() == [[1, 2], [3, -1], [-1, -1], [0, 4]]
    assert np.allclose(plain.route(l, 2, False)[1][3], [1 / 3, 1 / 3])


BAD = [dict(cols=0), dict(codes=0), dict(scales=0), dict(codes=SOME + 8), dict(scales=SOME + 4), dict(pitch=72), dict(pitch=48), dict(cols=0x7fffff01, pitch=0x80000000), dict(rows=0x7fffff01)]


@pytest.mark.parametrize("change", BAD)
def test_bad_matrices_are_refused(spg, lib, change):
    good, bad = _matrix(spg), _matrix(spg, **change)
    assert lib.spgk_fp8_quantize(SOME, 2, 64, 4, None, C.byref(bad), None) == -2
    assert b"spgk_fp8_quantize" in lib.spgk_error_string()
    assert lib.spgk_fp8_dequantize(C.byref(bad), SOME, 2, 64, None) == -2
    for w, x, nxt in ((bad, good, None), (good, bad, None), (good, good, bad)):
        n = None if nxt is None else C.byref(nxt)
        assert lib.spgk_layer_fp8(C.byref(w), None, 6, C.byref(x), SOME, 2, 64, n, SOME, None) == -2
        assert lib.spgk_experts_fp8(C.byref(w), 2, None, 6, C.byref(x), SOME, SOME, 2, 64, n, SOME, None) == -2


def test_bad_rows_are_refused(spg, lib):
    m = C.byref(_matrix(spg))
    for x, kind, ld in ((SOME, 3, 64), (SOME, -1, 64), (0, 2, 64), (SOME + 2, 2, 64), (SOME + 1, 0, 64), (SOME, 2, 63)):
        assert lib.spgk_fp8_quantize(x, kind, ld, 4, None, m, None) == -2, (x, kind, ld)
        assert lib.spgk_fp8_dequantize(m, x, kind, ld, None) == -2, (x, kind, ld)
    assert lib.spgk_fp8_quantize(SOME, 2, 64, 3, None, m, None) == -2                     # fewer rows than the matrix has
    assert lib.spgk_fp8_quantize(SOME, 2, 64, 4, SOME + 2, m, None) == -2 and lib.spgk_fp8_quantize(SOME, 2, 64, 0x80000001, SOME, m, None) == -2
    assert lib.spgk_fp8_quantize(SOME, 2, 64, 4, None, None, None) == -2
    huge = _matrix(spg, rows=0x7fffff00, cols=0x7fffff00, pitch=0x7fffff00)
    assert lib.spgk_fp8_quantize(SOME, 2, 0x7fffff00, 0x7fffff00, None, C.byref(huge), None) == -2
    none = C.byref(_matrix(spg, rows=0, codes=0, scales=0))
    assert lib.spgk_fp8_quantize(0, 2, 64, 0, None, none, None) == 0 and lib.spgk_fp8_dequantize(none, 0, 2, 64, None) == 0


def test_bad_layers_are_refused(spg, lib):
    w, x, other = _matrix(spg, rows=48), _matrix(spg), _matrix(spg, cols=96)

    def call(w=w, experts=None, bias=0, act=6, x=x, starts=SOME, y=SOME, kind=2, ldy=48, nxt=None, status=SOME):
        n = None if nxt is None else C.byref(nxt)
        if experts is None:
            return lib.spgk_layer_fp8(C.byref(w), bias, act, C.byref(x), y, kind, ldy, n, status, None)
        return lib.spgk_experts_fp8(C.byref(w), experts, bias, act, C.byref(x), starts, y, kind, ldy, n, status, None)
    for experts, out in ((None, 48), (3, 16)):
        nxt, wrong = _matrix(spg, cols=out), _matrix(spg, rows=5, cols=out)
        assert call(experts=experts, x=other) == -2 and call(experts=experts, w=_matrix(spg, rows=0)) == -2
        assert call(experts=experts, act=7) == -2 and call(experts=experts, act=-1) == -2 and call(experts=experts, y=0) == -2 and call(experts=experts, kind=3) == -2
        assert call(experts=experts, y=SOME + 2) == -2 and call(experts=experts, y=SOME + 1, kind=0) == -2
        assert call(experts=experts, ldy=out - 1) == -2 and call(experts=experts, status=0) == -2 and call(experts=experts, status=SOME + 2) == -2 and call(experts=experts, bias=SOME + 2) == -2
        wide = _matrix(spg, rows=3, cols=(1 << 27) + 32)
        assert call(experts=experts, w=wide, x=wide) == -2
        assert call(experts=experts, nxt=wrong) == -2 and call(experts=experts, nxt=other) == -2 and call(experts=experts, nxt=nxt, act=5) == -2
        assert call(experts=experts, x=_matrix(spg, rows=0)) == 0
    assert call(experts=0) == -2 and call(experts=1025) == -2 and call(experts=5) == -2 and call(experts=96) == -2
    assert call(experts=3, ldy=16, starts=0) == -2 and call(experts=3, ldy=16, starts=SOME + 2) == -2
    assert b"spgk_experts_fp8" in lib.spgk_error_string()


def test_bad_routes_are_refused(lib):
    def call(logits=SOME, kind=2, ld=10, n=2, experts=10, top=2, chosen=SOME, gates=2 * SOME, starts=3 * SOME, order=4 * SOME, places=5 * SOME):
        return lib.spgk_route_rows(logits, kind, ld, n, experts, top, 0, chosen, gates, starts, order, places, None)
    for bad in (dict(kind=3), dict(kind=-1), dict(experts=0), dict(experts=1025, ld=1025), dict(top=0), dict(top=11), dict(top=33, experts=64, ld=64), dict(logits=0), dict(chosen=0), dict(gates=0),
                dict(starts=0), dict(order=0), dict(places=0), dict(logits=SOME + 2), dict(logits=SOME + 1, kind=0), dict(ld=9), dict(chosen=SOME + 1), dict(gates=SOME + 2), dict(starts=SOME + 2),
                dict(order=SOME + 2), dict(places=SOME + 3), dict(n=1 << 29), dict(n=0, starts=0),
                dict(places=SOME), dict(order=2 * SOME), dict(starts=5 * SOME)):
        assert call(**bad) == -2, bad
        assert b"spgk_route_rows" in lib.spgk_error_string()


def test_bad_sums_are_refused(lib):
    def call(y=SOME, kind=2, ldy=10, y_rows=8, places=SOME, gates=SOME, n=4, top=2, width=10, out=SOME, out_kind=2, ldo=10):
        return lib.spgk_combine_rows(y, kind, ldy, y_rows, places, gates, n, top, width, out, out_kind, ldo, None)
    for bad in (dict(kind=3), dict(out_kind=3), dict(kind=-1), dict(top=0), dict(width=0), dict(y=0), dict(places=0), dict(gates=0), dict(out=0), dict(y=SOME + 2), dict(out=SOME + 2), dict(out=SOME + 1, out_kind=1),
                dict(places=SOME + 2), dict(gates=SOME + 2), dict(y_rows=0x80000001), dict(ldy=9), dict(ldo=9)):
        assert call(**bad) == -2, bad
        assert b"spgk_combine_rows" in lib.spgk_error_string()
    assert call(n=0) == 0
