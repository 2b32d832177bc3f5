"""Layers on microscaled operands whose waits give up with copies and products under way: what was not summed is not put out, and the next call is sound."""
import ctypes as C

import numpy as np
import pytest

import mx4_plain as plain
from test_gpu_mx4 import Packed, _dtype, _random, lib  # noqa: F401  (lib: fixture)

pytestmark = pytest.mark.gpu

TIMEOUT = -4
PAIRS = 74                                                   # of 148 SMs
SINGLE = [(1, 784, 512), (1, 200, 60), (3, 1000, 16384), (16, 130, 8192), (64, 8192, 1000), (100, 260, 2048), (60, 40000, 64), (128, 512, 784)]
IN_PAIRS = [(200, 30000, 64), (2500, 2700, 300), (4100, 1100, 70), (3001, 5003, 1800), (300, 30000, 1601), (9000, 1700, 2100)]


class Call:
    """A layer with fp32 or 16-bit rows and a next operand as its outputs."""

    def __init__(self, spg, lib, n, out, k, t):
        import torch
        rng = np.random.default_rng(n + out + k)
        self.lib, self.n, self.out, self.t = lib, n, out, t
        (self.w, self.wv), (self.x, self.xv) = _random(spg, out, k, rng, True), _random(spg, n, k, rng, True)
        self.y = torch.empty((n, out), dtype=_dtype(t), device="cuda")
        self.next = Packed(spg, n, out)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self, impatient):
        """(status call's answer, rows, the next operand's codes and scale tiles); what is not written is NaN, 0xA5 and 0xFF"""
        self.y.fill_(float("nan"))
        self.next.codes.fill_(0xA5)
        self.next.tiles.fill_(0xFF)
        self.lib.spgk_selftest_impatient(int(impatient))
        try:
            assert self.lib.spgk_layer_mx4(self.w.ref, None, 6, self.x.ref, self.y.data_ptr(), self.t, self.out, self.next.ref, self.status.data_ptr(), None) == 0, self.lib.spgk_error_string()
        finally:
            self.lib.spgk_selftest_impatient(0)
        rc = self.lib.spgk_gemm_tc_status(self.status.data_ptr(), None)
        return rc, self.y.float().cpu().numpy(), self.next.codes.cpu().numpy(), self.next.tiles.cpu().numpy()

    def right(self, y):
        """The sums are whole multiples of 1/16 below 2^19: exact, but for the one rounding of the output."""
        import torch
        want = torch.from_numpy(self.xv).cuda() @ torch.from_numpy(self.wv).cuda().T
        return np.array_equal(y, want.to(_dtype(self.t)).float().cpu().numpy())


@pytest.mark.parametrize("n,out,k", SINGLE)
def test_nothing_is_put_out_by_a_tile_that_was_given_up(spg, lib, n, out, k):
    c = Call(spg, lib, n, out, k, 2)
    for _ in range(2):
        rc, y, codes, tiles = c.run(True)
        assert rc == TIMEOUT and b"bounded wait 2 " in lib.spgk_error_string()
        assert np.isnan(y).all() and (codes == 0xA5).all() and (tiles == 0xFF).all()
        rc, y, codes, tiles = c.run(False)
        assert rc == 0, lib.spgk_error_string()
        assert c.right(y) and not (tiles[:512] == 0xFF).all()


@pytest.mark.parametrize("n,out,k", IN_PAIRS)
@pytest.mark.parametrize("t", [2, 1])
def test_a_pair_gives_up_its_last_tile_alone(spg, lib, n, out, k, t):
    """Every pair gives up its last tile of 256 x 256: that is left alone in both of its CTAs, all others are right."""
    c = Call(spg, lib, n, out, k, t)
    for _ in range(2):
        rc, y, codes, tiles = c.run(False)
        assert rc == 0 and c.right(y)
        rc, y1, codes1, tiles1 = c.run(True)
        assert rc == TIMEOUT and b"bounded wait 2 " in lib.spgk_error_string()
        left = np.zeros((-(-n // 256), -(-out // 256)), bool)
        for r in range(left.shape[0]):
            for j in range(left.shape[1]):
                rows, units = slice(256 * r, min(n, 256 * r + 256)), slice(256 * j, min(out, 256 * j + 256))
                held = slice(128 * j, -(-units.stop // 32) * 16)
                blocks = np.arange(8 * j, -(-units.stop // 32))
                at = plain.scale_place(out, np.arange(rows.start, rows.stop)[:, None], blocks[None])
                left[r, j] = np.isnan(y1[rows, units]).all()
                if left[r, j]:
                    assert (codes1[rows, held] == 0xA5).all() and (tiles1[at] == 0xFF).all()
                else:
                    assert np.array_equal(y1[rows, units], y[rows, units])
                    assert np.array_equal(codes1[rows, held], codes[rows, held]) and np.array_equal(tiles1[at], tiles[at])
        assert left.sum() == min(PAIRS, left.size)


def test_products_do_not_take_the_place_of_sums_that_are_not_taken_yet(spg, lib):
    """Pairs of seven short tiles that give up the wait for tensor memory where the sums of the tile before still lie there: what is put out is right, the rest is left alone."""
    import torch
    n, out, k = 4096, 8192, 512
    w, x = Packed(spg, out, k), Packed(spg, n, k)
    for m in (w, x):
        m.codes.random_()
        m.tiles.fill_(127)
    y = torch.empty((n, out), dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(impatient):
        y.fill_(float("nan"))
        lib.spgk_selftest_impatient(impatient)
        try:
            assert lib.spgk_layer_mx4(w.ref, None, 6, x.ref, y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0
        finally:
            lib.spgk_selftest_impatient(0)
        return lib.spgk_gemm_tc_status(status.data_ptr(), None), y.clone()
    rc, right = run(0)
    assert rc == 0 and right.isfinite().all()
    for _ in range(3):
        rc, got = run(2)
        assert rc == TIMEOUT and b"bounded wait 6 " in lib.spgk_error_string()
        put = got.isfinite()
        assert 0 < int(put.sum()) < n * out
        assert torch.equal(got[put], right[put])
    rc, got = run(0)
    assert rc == 0 and torch.equal(got, right)
