"""Layers on 8-bit operands whose waits give up with copies and products under way: what was not summed is not put out, and the next call is sound."""
import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_fp8 import Packed, _dtype, _random, lib  # noqa: F401  (lib: fixture)

pytestmark = pytest.mark.gpu

TIMEOUT = -4


class Call:
    """A layer, or one for each group of rows, with rows and a next operand as its outputs."""

    def __init__(self, spg, lib, n, out, k, starts=None, t=2):
        import torch
        rng = np.random.default_rng(n + out + k)
        self.lib, self.n, self.out, self.t, self.experts = lib, n, out, t, 1 if starts is None else len(starts) - 1
        (self.w, self.wv), (self.x, self.xv) = _random(spg, out * self.experts, k, rng, True), _random(spg, n, k, rng, True)
        self.starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.groups = [(0, n)] if starts is None else plain.ranges(starts, n)
        self.y = torch.empty((n, out), dtype=_dtype(t), device="cuda")
        self.next = Packed(spg, n, out)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self, impatient):
        """(status call's answer, rows, the next operand's codes and scales); what is not written is NaN, 0xA5 and 0xFF"""
        self.y.fill_(float("nan"))
        self.next.codes.fill_(0xA5)
        self.next.words.fill_(0xFF)
        self.lib.spgk_selftest_impatient(impatient)
        try:
            if self.starts is None:
                rc = self.lib.spgk_layer_fp8(self.w.ref, None, 6, self.x.ref, self.y.data_ptr(), self.t, self.out, self.next.ref, self.status.data_ptr(), None)
            else:
                rc = self.lib.spgk_experts_fp8(self.w.ref, self.experts, None, 6, self.x.ref, self.starts.data_ptr(), self.y.data_ptr(), self.t, self.out, self.next.ref, self.status.data_ptr(), None)
            assert rc == 0, self.lib.spgk_error_string()
        finally:
            self.lib.spgk_selftest_impatient(0)
        rc = self.lib.spgk_gemm_tc_status(self.status.data_ptr(), None)
        code, scale = self.next.host()
        return rc, self.y.float().cpu().numpy(), code, scale

    def want(self):
        """The sums are whole multiples of 1/64 below 2^18: exact, but for the one rounding of the output."""
        import torch
        x, w = torch.from_numpy(self.xv).cuda(), torch.from_numpy(self.wv).cuda()
        y = torch.full((self.n, self.out), float("nan"), dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(self.groups):
            y[lo:hi] = x[lo:hi] @ w[e * self.out:(e + 1) * self.out].T
        return y.to(_dtype(self.t)).float().cpu().numpy()


ALL = [(1, 784, 512, None), (1, 200, 60, None), (3, 1000, 16384, None), (16, 130, 8192, None), (64, 4000, 1000, None), (100, 260, 2048, None), (128, 512, 784, None),
       (7, 300, 777, [0, 1, 2, 2, 7]), (40, 200, 4096, [3, 10, 10, 33])]


@pytest.mark.parametrize("n,out,k,starts", ALL)
def test_nothing_is_put_out_by_tiles_that_were_given_up(spg, lib, n, out, k, starts):
    c = Call(spg, lib, n, out, k, starts)
    want = c.want()
    for _ in range(2):
        rc, y, code, scale = c.run(1)
        assert rc == TIMEOUT and b"bounded wait 2 " in lib.spgk_error_string()
        assert np.isnan(y).all() and (code == 0xA5).all() and (scale == 0xFF).all()
        rc, y, code, scale = c.run(0)
        assert rc == 0, lib.spgk_error_string()
        assert np.array_equal(y, want, equal_nan=True)


SOME = [(200, 30000, 64, None), (2500, 2700, 300, None), (4100, 1100, 70, None), (3001, 5003, 1800, None), (300, 30000, 1601, None), (9000, 1700, 2100, None), (60, 40000, 64, None),
        (3000, 2000, 400, [0, 7, 900, 900, 2600, 3000]), (500, 3000, 300, list(range(0, 501, 10))), (6000, 2100, 520, [0, 3100, 6000])]


@pytest.mark.parametrize("n,out,k,starts", SOME)
@pytest.mark.parametrize("t", [2, 1])
def test_the_last_tiles_alone_are_given_up(spg, lib, n, out, k, starts, t):
    """Every CTA, or pair, gives up its last tile: that is left alone whole, all others are right."""
    c = Call(spg, lib, n, out, k, starts, t)
    want = c.want()
    rc, y, code, scale = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)
    for _ in range(2):
        rc, y1, code1, scale1 = c.run(1)
        assert rc == TIMEOUT and b"bounded wait 2 " in lib.spgk_error_string()
        left = np.isnan(y1)
        inside = ~np.isnan(want)
        assert 0 < (left & inside).sum() < inside.sum()
        assert np.array_equal(y1[~left], y[~left])
        blocks = plain.blocks(out)
        whole = np.pad(left, ((0, 0), (0, -out % 128)), mode="edge").reshape(n, blocks, 128)
        assert (whole.all(-1) == whole.any(-1)).all()             # (a row's units of a tile go together)
        gone = whole.all(-1)
        assert (scale1[gone] == 0xFF).all() and np.array_equal(scale1[~gone], scale[~gone])
        cols = np.repeat(gone, 128, 1)[:, :out]
        assert (code1[cols] == 0xA5).all() and np.array_equal(code1[~cols], code[~cols])
    rc, y, *_ = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)


@pytest.mark.parametrize("n,out,k,starts", [(4096, 8192, 512, None), (64, 60000, 128, None), (4096, 4096, 256, [0, 1000, 1001, 4096])])
def test_products_do_not_take_the_place_of_sums_that_are_not_taken_yet(spg, lib, n, out, k, starts):
    """Short tiles, several a CTA or pair, that give up the wait for tensor memory where the sums of a tile before still lie there: what is put out is right."""
    c = Call(spg, lib, n, out, k, starts)
    want = c.want()
    rc, y, *_ = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)
    for _ in range(3):
        rc, y, *_ = c.run(2)
        put = np.isfinite(y)
        assert rc in (0, TIMEOUT) and np.array_equal(y[put], want[put])
        assert rc == 0 or 0 < put.sum() < y.size
    rc, y, *_ = c.run(0)
    assert rc == 0 and np.array_equal(y, want, equal_nan=True)
