"""Layers on 8-bit operands that give up the wait for room in tensor memory, and are seen to: the sums that lie there are put out right, or a tile is left alone whole."""
import numpy as np
import pytest

from test_gpu_fp8 import lib  # noqa: F401  (fixture)
from test_gpu_fp8_waits import TIMEOUT, Call

pytestmark = pytest.mark.gpu


# Short tiles, several a CTA or pair, whose products are done long before the outputs of the tile before; and long sums, whose chains follow one another in one tile.  Of pairs they have columns in
# common, which cannot be taken yet when the last product before them is only under way.  CTAs of their own have room for two chains, and the one before the last may have been taken by then.
CASES = [(64, 60000, 128, None), (120, 60000, 128, None), (16, 80000, 128, None), (4096, 8192, 512, None), (4096, 4096, 256, [0, 1000, 1001, 4096]), (600, 9000, 128, [0, 0, 300, 600]),
         (4096, 8192, 4096, None), (1000, 2600, 9000, None), (500, 1300, 6000, [0, 10, 500])]


@pytest.mark.parametrize("n,out,k,starts", CASES)
def test_rooms_that_are_not_free_yet_are_seen(spg, lib, n, out, k, starts):
    c = Call(spg, lib, n, out, k, starts)
    want = c.want()
    rc, y, code, scale = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)
    gave_up = 0
    for _ in range(5):
        rc, y1, code1, scale1 = c.run(2)
        assert rc in (0, TIMEOUT)
        if rc == TIMEOUT:
            gave_up += 1
            assert b"bounded wait 6 " in lib.spgk_error_string()
            assert np.isnan(y1[~np.isnan(want)]).any()            # (some tile was left alone)
        put = ~np.isnan(y1)
        assert np.array_equal(y1[put], y[put])
        # a row's units of a tile, and the block of the next operand that they are, were put out whole or not at all
        whole = np.pad(put, ((0, 0), (0, -out % 128)), mode="edge").reshape(n, -1, 128)
        assert (whole.all(-1) == whole.any(-1)).all()
        there = whole.all(-1)
        assert (scale1[~there] == 0xFF).all() and np.array_equal(scale1[there], scale[there])
    assert gave_up > 0 or (n, k) == (500, 6000)
    rc, y, *_ = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)
