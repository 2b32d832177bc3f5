"""How far sums of layers on 8-bit operands may be off, at lengths and in arrangements (one CTA a tile, several, pairs) where losses add up."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_fp8 import lib  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu

ONE = 56                                                          # the code of 1; the seven behind it are 1.125 to 1.875


class Matrix:
    """Codes [rows][cols] on the device, and a scale byte for each block, [rows][blocks]."""

    def __init__(self, spg, code, scale):
        import torch
        rows, cols = code.shape
        self.code, self.scale, self.pitch = code, scale, -(-cols // 16) * 16
        self.codes = torch.zeros((rows, self.pitch), dtype=torch.uint8, device="cuda")
        self.codes[:, :cols] = code
        groups = -(-scale.shape[1] // 4)
        self.words = torch.full((groups, rows, 4), 0xFF, dtype=torch.uint8, device="cuda")
        for b in range(scale.shape[1]):
            self.words[b // 4, :, b % 4] = scale[:, b]
        self.m = spg.abi.Fp8(self.codes.data_ptr(), self.words.data_ptr(), rows, cols, self.pitch)

    def values(self, lo, hi, a, b):
        """Rows lo to hi, columns a to b (a: a block's first), in 64 bits."""
        import torch
        size = torch.from_numpy(np.concatenate([plain.SIZES, -plain.SIZES])).cuda()
        v = size[self.code[lo:hi, a:b].int()]
        s = torch.exp2(self.scale[lo:hi, a // plain.BLOCK:-(-b // plain.BLOCK)].double() - 127)
        return v * s.repeat_interleave(plain.BLOCK, 1)[:, :b - a]


def _codes(rows, cols, seed, signs):
    """1 to 1.875, of both signs or one"""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    code = torch.randint(ONE, ONE + 8, (rows, cols), device="cuda", generator=g, dtype=torch.uint8)
    if signs:
        code |= torch.randint(0, 2, (rows, cols), device="cuda", generator=g, dtype=torch.uint8) << 7
    return code


def _scales(rows, cols, byte=127):
    import torch
    return torch.full((rows, plain.blocks(cols)), byte, dtype=torch.uint8, device="cuda")


def _run(spg, lib, w, x, out, starts=None):
    """(what came, sums in 64 bits, sums of magnitudes)"""
    import torch
    n, k = x.code.shape
    experts = 1 if starts is None else len(starts) - 1
    y = torch.zeros((n, out), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    if starts is None:
        assert lib.spgk_layer_fp8(C.byref(w.m), None, 6, C.byref(x.m), y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0, lib.spgk_error_string()
    else:
        at = torch.tensor(starts, dtype=torch.int32, device="cuda")
        assert lib.spgk_experts_fp8(C.byref(w.m), experts, None, 6, C.byref(x.m), at.data_ptr(), y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0, lib.spgk_error_string()
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    want, size = torch.zeros((n, out), dtype=torch.float64, device="cuda"), torch.zeros((n, out), dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate([(0, n)] if starts is None else plain.ranges(starts, n)):
        for j in range(0, out if hi > lo else 0, 1024):
            end = min(out, j + 1024)
            for a in range(0, k, 32768):
                wv, xv = w.values(e * out + j, e * out + end, a, min(k, a + 32768)), x.values(lo, hi, a, min(k, a + 32768))
                want[lo:hi, j:end] += xv @ wv.T
                size[lo:hi, j:end] += xv.abs() @ wv.abs().T
    return y.double(), want, size


# one CTA a tile of 16, 64 and 128 rows (more tiles than two CTAs each find room for), eight and two CTAs a tile, pairs; groups
LONG = [(1, 9700, 16384, None), (60, 9700, 16384, None), (120, 9700, 16384, None), (1, 128, 65536, None), (100, 4000, 16384, None), (700, 2600, 16384, None), (300, 520, 65536, None), (3000, 1000, 20000, None),
        (40, 3000, 16384, [0, 1, 30, 40]), (700, 1300, 16384, [0, 1, 320, 700])]


@pytest.mark.parametrize("n,out,k,starts", LONG)
def test_long_sums_of_one_sign(spg, lib, n, out, k, starts):
    """Products are whole multiples of 2^-11 (those of every other block; of 2^-6 in the rest) below 4, so sums over up to 24 blocks, half of them of each kind, lie below 1.5 * (2^12 + 2^7) < 2^13 and are
    exact in the 24 bits that the tensor core keeps; those of a layer are not.  24 blocks at most follow one another there, and four at least but for the ends of a CTA's part, of which there are eight at most.
    Their sums are added up rounding to nearest, half of 2^-23 of the sum at most each time: no more than 2^-24 of the result for each addition."""
    import torch
    experts = 1 if starts is None else len(starts) - 1
    scale = _scales(experts * out, k)
    odd = (torch.arange(scale.shape[0], device="cuda")[:, None] + torch.arange(scale.shape[1], device="cuda")[None]) % 2
    w, x = Matrix(spg, _codes(experts * out, k, n + k, False), scale - 5 * odd.to(torch.uint8)), Matrix(spg, _codes(n, k, n, False), _scales(n, k))
    got, want, size = _run(spg, lib, w, x, out, starts)
    assert want.max() > 2.0 ** 13.5                               # (in units of 2^-11: beyond 24 bits)
    additions = -(-k // 512) + 16
    off = ((got - want).abs() / want.clamp_min(1)).max().item()
    assert off <= additions * 2.0 ** -24, off * 2.0 ** 24 / additions


@pytest.mark.parametrize("n,out,k,starts", LONG + [(1, 16384, 8192, None), (64, 1030, 8200, None), (200, 8192, 8192, None), (1000, 2048, 8192, None), (65, 300, 70001, None), (5, 640, 30000, [0, 2, 2, 5])])
def test_long_dense_sums_that_need_no_rounding(spg, lib, n, out, k, starts):
    """No element is zero; whole multiples of 1/64 whose magnitudes come to less than 3.52 k, below 2^18: exact in any order and any cut.  One product left out, or taken twice, is 1 at least."""
    experts = 1 if starts is None else len(starts) - 1
    w, x = Matrix(spg, _codes(experts * out, k, n * 2 + k, True), _scales(experts * out, k)), Matrix(spg, _codes(n, k, n + 1, True), _scales(n, k))
    got, want, size = _run(spg, lib, w, x, out, starts)
    assert size.max() < 2.0 ** 18
    assert (got == want).all()


@pytest.mark.parametrize("n,out,k,starts", [s for s in LONG if s[2] <= 20000] + [(1, 128, 8192, None), (1, 16384, 8192, None), (1, 1000, 16384, None), (100, 2000, 8192, None), (512, 8192, 8192, None), (24, 700, 8192, [0, 3, 24])])
@pytest.mark.parametrize("signs", [True, False])
def test_long_sums_of_any_elements(spg, lib, signs, n, out, k, starts):
    """Elements of all sizes, scales of 1/4 to 4.  An addition has 33 numbers, each of which may lose what lies below 2^-24 of the largest, itself no larger than the sum of all magnitudes
    of its chain; a chain has 96 additions at most, however long the sum is; the chains (see above) are added up rounding to nearest.  A block left out is seen."""
    import torch
    experts = 1 if starts is None else len(starts) - 1
    g = torch.Generator(device="cuda")
    g.manual_seed(n + out + k)

    def matrix(rows):
        code = torch.randint(0, 127, (rows, k), device="cuda", generator=g, dtype=torch.uint8)
        if signs:
            code |= torch.randint(0, 2, (rows, k), device="cuda", generator=g, dtype=torch.uint8) << 7
        return Matrix(spg, code, torch.randint(125, 130, (rows, plain.blocks(k)), device="cuda", generator=g, dtype=torch.uint8))
    w, x = matrix(experts * out), matrix(n)
    got, want, size = _run(spg, lib, w, x, out, starts)
    tol = (96 * 33 + -(-k // 512) + 16) * 2.0 ** -24 * size
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / size.clamp_min(1e-30)).max().item() * 2.0 ** 24
    if starts is None:
        for b in (0, plain.blocks(k) // 2, plain.blocks(k) - 1):
            lo, hi = b * plain.BLOCK, min(k, (b + 1) * plain.BLOCK)
            part = x.values(0, n, lo, hi) @ w.values(0, out, lo, hi).T
            assert ((got - (want - part)).abs() > tol).any()
