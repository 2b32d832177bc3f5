"""8-bit numbers in blocks of 128 on the GPU: quantising and back byte for byte, layers for all rows and by groups of them against sums in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain as plain

pytestmark = pytest.mark.gpu

HALF = {0: 2.0 ** -11, 1: 2.0 ** -8, 2: 2.0 ** -24}       # half a step of fp16, bf16, fp32


@pytest.fixture(scope="module")
def lib(spg, has_gpu):
    assert has_gpu, "no CUDA device"
    return spg.lib()


def _dtype(t):
    import torch
    return {0: torch.float16, 1: torch.bfloat16, 2: torch.float32}[t]


class Packed:
    """A matrix on the device, with what it points to; a row and 16 bytes of scales more than it has."""

    def __init__(self, spg, rows, cols, code=None, scale=None, more=0):
        import torch
        self.rows, self.cols, self.pitch = rows, cols, -(-cols // 16) * 16 + more
        self.codes = torch.full((rows + 1, self.pitch), 0xA5, dtype=torch.uint8, device="cuda")
        self.words = torch.full((-(-plain.blocks(cols) // 4) * rows * 4 + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        if code is not None:
            c, w = plain.pack(code, scale, self.pitch, 0xFF)      # (NaN in what is not looked at)
            self.codes[:rows] = torch.from_numpy(c).cuda()
            self.words[:-16] = torch.from_numpy(w).cuda()
        self.m = spg.abi.Fp8(self.codes.data_ptr(), self.words.data_ptr(), rows, cols, self.pitch)
        self.ref = C.byref(self.m)

    def host(self):
        return plain.unpack(self.codes.cpu().numpy(), self.words.cpu().numpy(), self.rows, self.cols)


def _random(spg, rows, cols, rng, exact=False, more=0):
    """Random codes and scales; exact: whole multiples of 1/4 up to 8, for sums without rounding."""
    if exact:
        code = rng.choice(np.flatnonzero((plain.SIZES[:127] <= 8) & (plain.SIZES[:127] * 4 % 1 == 0)), (rows, cols)).astype(np.uint8)
        code |= (rng.integers(0, 2, code.shape) << 7).astype(np.uint8)
        scale = rng.integers(126, 129, (rows, plain.blocks(cols)))
    else:
        code = rng.integers(0, 254, (rows, cols)).astype(np.uint8)
        code[code >= 127] += 1                                   # every code but the two NaN
        scale = rng.integers(110, 128, (rows, plain.blocks(cols)))
    scale = scale.astype(np.uint8)
    return Packed(spg, rows, cols, code, scale, more), plain.values(code, scale)


def _values_with_extremes(rows, cols, t, rng):
    import torch
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    x.reshape(-1)[:: 37] = 0.0
    if rows > 2:
        x[1] = 0.0                                               # a row of zeros
        x[2, : cols // 2] *= 2.0 ** -140                         # far below the smallest scale
    if rows > 5:
        x[3] = np.resize([448, 17, 19, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 2.0 ** -9, 232, -17, -19, -1.0625, -2.0 ** -10, -448, 9.5], cols)   # half way
        x[4, :: 3] = -0.0
        x[5, cols // 2] = np.nan
    if rows > 7:
        x[6, 0] = np.inf
        x[7, cols - 1] = -np.inf
    if rows > 8 and t != 0:
        x[8] = np.resize([3.3e38, -1e38, 1e-44, 2.0 ** -126, 3.0 * 2.0 ** -127], cols)
    if rows > 9:
        x[9] *= 448.5 / np.abs(x[9]).max()                       # next to the largest a scale has room for
    return torch.from_numpy(x.astype(np.float32)).to(_dtype(t))


@pytest.mark.parametrize("t", [2, 1, 0])
@pytest.mark.parametrize("rows,cols,pad,off", [(1, 1, 0, 0), (1, 8192, 0, 0), (9, 127, 0, 0), (9, 128, 0, 0), (10, 129, 3, 0), (130, 777, 24, 0), (257, 513, 1, 1), (12, 1000, 0, 3), (300, 256, 8, 8), (64, 4100, 4, 0)])
def test_quantize_and_back(spg, lib, t, rows, cols, pad, off):
    import torch
    rng = np.random.default_rng(rows * 1000 + cols + t)
    x = _values_with_extremes(rows, cols, t, rng)
    buf = torch.zeros(rows * (cols + pad) + off, dtype=x.dtype, device="cuda")
    view = buf[off:].view(rows, cols + pad)
    view[:, :cols] = x.cuda()
    view[:, cols:] = float("nan")                                # what is beside a row is not read
    m = Packed(spg, rows, cols, more=16 if pad else 0)
    assert lib.spgk_fp8_quantize(view.data_ptr(), t, cols + pad, rows, None, m.ref, None) == 0, lib.spgk_error_string()
    torch.cuda.synchronize()
    want_code, want_scale = plain.quantize(x.double().numpy())
    code, scale = m.host()
    assert np.array_equal(scale, want_scale)
    assert np.array_equal(code, want_code)
    codes, words = m.codes.cpu().numpy(), m.words.cpu().numpy()
    assert (codes[rows] == 0xA5).all() and (words[-16:] == 0xFF).all() and (codes[:, -(-cols // 16) * 16:] == 0xA5).all()
    want = plain.values(want_code, want_scale)
    for to in (2, 1, 0):
        y = torch.full((rows + 1, cols + pad), 7.0, dtype=_dtype(to), device="cuda")
        assert lib.spgk_fp8_dequantize(m.ref, y.data_ptr(), to, cols + pad, None) == 0, lib.spgk_error_string()
        got = y.cpu()
        assert (got[rows] == 7).all() and (got[:, cols:] == 7).all()
        expect = torch.from_numpy(want).float().to(_dtype(to))
        assert torch.equal(torch.nan_to_num(got[:rows, :cols], 12345.0), torch.nan_to_num(expect, 12345.0))
        assert torch.equal(torch.isnan(got[:rows, :cols]), torch.isnan(expect))


@pytest.mark.parametrize("t,cols,pad", [(2, 777, 3), (1, 1024, 0), (0, 130, 6)])
def test_quantize_takes_rows_by_index(spg, lib, t, cols, pad):
    """The same row twice, none of x's rows (below zero and beyond the last): zeros."""
    import torch
    rng = np.random.default_rng(cols)
    x = _values_with_extremes(11, cols, t, rng)
    full = torch.full((11, cols + pad), float("nan"), dtype=x.dtype, device="cuda")
    full[:, :cols] = x.cuda()
    index = torch.tensor([3, 3, 10, 0, -1, 11, 5, -2 ** 31, 2 ** 31 - 1, 7, 8, 9, 9], dtype=torch.int32, device="cuda")
    m = Packed(spg, len(index), cols)
    assert lib.spgk_fp8_quantize(full.data_ptr(), t, cols + pad, 11, index.data_ptr(), m.ref, None) == 0, lib.spgk_error_string()
    torch.cuda.synchronize()
    src = x.double().numpy()
    want = np.stack([src[i] if 0 <= i < 11 else np.zeros(cols) for i in index.tolist()])
    code, scale = m.host()
    want_code, want_scale = plain.quantize(want)
    assert np.array_equal(scale, want_scale) and np.array_equal(code, want_code)
    none = Packed(spg, 3, cols)
    assert lib.spgk_fp8_quantize(None, t, cols + pad, 0, index.data_ptr(), none.ref, None) == 0
    torch.cuda.synchronize()
    code, scale = none.host()
    assert (code == 0).all() and (scale == 0).all()


SHAPES = [(1, 1, 1), (1, 10, 1000), (2, 333, 777), (16, 128, 128), (17, 129, 31), (33, 300, 64), (65, 257, 1025), (128, 512, 784), (300, 1000, 512), (513, 130, 4100), (600, 64, 33),
          (1, 128, 16384), (8, 200, 8192), (40, 96, 3001), (700, 1500, 320), (129, 1, 200), (257, 2, 40), (2500, 2700, 300), (4100, 1100, 70), (90, 33, 20000),
          (9, 900, 2048), (24, 130, 4096), (64, 1030, 4096), (100, 260, 2048), (128, 1100, 1024), (300, 390, 4096), (1, 2100, 640), (3, 19000, 129)]


class Call:
    """A layer, or one for each group of rows, and what it has to give."""

    def __init__(self, spg, lib, rng, n, out, k, starts=None, exact=False, bias=True):
        import torch
        self.lib, self.spg, self.n, self.out, self.k = lib, spg, n, out, k
        self.experts = 1 if starts is None else len(starts) - 1
        self.w, self.wv = _random(spg, out * self.experts, k, rng, exact)
        self.x, self.xv = _random(spg, n, k, rng, exact, more=32 if n % 2 else 0)
        self.b = (rng.integers(-8, 9, out * self.experts) if exact else rng.standard_normal(out * self.experts)).astype(np.float32) * (1 if bias else 0)
        self.bd = torch.from_numpy(self.b).cuda() if bias else None
        self.starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.groups = [(0, n)] if starts is None else plain.ranges(starts, n)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self, act, y=None, t=2, ldy=0, nxt=None, stream=None):
        y = None if y is None else y.data_ptr()
        b = None if self.bd is None else self.bd.data_ptr()
        n = None if nxt is None else nxt.ref
        if self.starts is None:
            rc = self.lib.spgk_layer_fp8(self.w.ref, b, act, self.x.ref, y, t, ldy, n, self.status.data_ptr(), stream)
        else:
            rc = self.lib.spgk_experts_fp8(self.w.ref, self.experts, b, act, self.x.ref, self.starts.data_ptr(), y, t, ldy, n, self.status.data_ptr(), stream)
        assert rc == 0, self.lib.spgk_error_string()
        assert self.lib.spgk_gemm_tc_status(self.status.data_ptr(), stream) == 0, self.lib.spgk_error_string()

    def rows(self, act, t, gap=0):
        """(what came, [rows][out]; what is beside and behind is checked to be as it was)"""
        import torch
        ldy = self.out + gap
        y = torch.full((self.n + 1, ldy), -3.0, dtype=_dtype(t), device="cuda")
        self.run(act, y, t, ldy)
        got = y.double().cpu().numpy()
        assert (got[self.n] == -3).all() and (got[:, self.out:] == -3).all()
        return got[:self.n, :self.out]

    def want(self, act):
        """(values, sums of magnitudes) in 64 bits; -3 where no group has the row"""
        import torch
        v, size = np.full((self.n, self.out), -3.0), np.zeros((self.n, self.out))
        for e, (lo, hi) in enumerate(self.groups):
            if hi <= lo:
                continue
            w, b, x = self.wv[e * self.out:(e + 1) * self.out], self.b[e * self.out:(e + 1) * self.out].astype(float), self.xv[lo:hi]
            wd, xd = torch.from_numpy(w).cuda(), torch.from_numpy(x).cuda()
            with np.errstate(over="ignore"):
                v[lo:hi] = plain.ACTS[act]((xd @ wd.T).cpu().numpy() + b)
            size[lo:hi] = (xd.abs() @ wd.abs().T).cpu().numpy() + np.abs(b)
        return v, size

    def tolerance(self, want, size, t):
        # A step adds 32 products to the sum: 33 numbers, of which each may lose what lies below 2^-24 of the largest, itself no larger than the sum of
        # all magnitudes; then the bias, the activation (no steeper than 1; 4 ulp of its own functions) and the rounding of the output.
        steps = -(-self.k // 32) + 1
        return steps * 33 * 2.0 ** -24 * size + np.abs(want) * (HALF[t] + 4 * 2.0 ** -23) + (2.0 ** -25 if t == 0 else 0)


def _close(got, want, tol, t):
    big = np.abs(want) > 65504
    if t == 0:
        assert np.all(np.isinf(got[big]) | (np.abs(got[big]) >= 65000))
        got, want, tol = got[~big], want[~big], tol[~big]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want)[bad].max()), float(tol[bad].min()))


@pytest.mark.parametrize("n,out,k", [s for s in SHAPES if s[2] <= 4100])          # (longer sums would need more bits)
def test_layer_sums_that_need_no_rounding(spg, lib, n, out, k):
    """Whole multiples of 1/64 below 2^18: every sum is exact in 32 bits, whatever its order."""
    c = Call(spg, lib, np.random.default_rng(n + out + k), n, out, k, exact=True)
    assert np.abs(c.want(6)[1]).max() < 2.0 ** 18
    assert np.array_equal(c.rows(6, 2, n % 3), c.want(6)[0])


@pytest.mark.parametrize("n,out,k", SHAPES)
@pytest.mark.parametrize("t", [2, 1, 0])
def test_layer_against_64_bits(spg, lib, n, out, k, t):
    act = (n + out + k + t) % 7
    c = Call(spg, lib, np.random.default_rng(n * 3 + out + k), n, out, k, bias=(n + t) % 4 != 0)
    want, size = c.want(act)
    _close(c.rows(act, t, n % 3), want, c.tolerance(want, size, t), t)


def _starts(rng, n, experts, some=1.0):
    """Random groups of n rows in all, a share of them without rows."""
    share = rng.random(experts) * (rng.random(experts) < some) + 1e-9
    return np.concatenate(([0], np.cumsum(rng.multinomial(n, share / share.sum()))))


GROUPS = [(1, 40, 100, [0, 1]), (1, 40, 100, [0, 0, 1, 1]), (5, 130, 300, [0, 0, 0, 0]), (7, 300, 777, [0, 1, 2, 2, 7]), (40, 200, 260, [3, 10, 10, 33]), (64, 129, 1000, None), (200, 500, 129, None),
          (333, 257, 640, None), (1500, 300, 513, None), (3000, 1000, 384, None), (4000, 600, 200, None), (128, 64, 4096, [0, 128]), (700, 900, 256, [0, 1, 700]), (600, 128, 128, [0, 255, 256, 513, 600]),
          (2000, 1111, 300, [0, 0, 1999, 2000, 2000])]


@pytest.mark.parametrize("n,out,k,starts", GROUPS)
@pytest.mark.parametrize("t", [2, 1])
def test_experts_against_64_bits(spg, lib, n, out, k, starts, t):
    rng = np.random.default_rng(n + out * 3 + k)
    if starts is None:
        starts = _starts(rng, n, 3 + n % 14, 0.7)
    act = (n + t) % 7
    c = Call(spg, lib, rng, n, out, k, starts, bias=n % 3 != 0)
    want, size = c.want(act)
    got = c.rows(act, t, n % 2)
    none = np.ones(n, bool)
    for lo, hi in c.groups:
        none[lo:hi] = False
    assert (got[none] == -3).all()                                # rows of no group are as they were
    _close(got[~none], want[~none], c.tolerance(want, size, t)[~none], t)


@pytest.mark.parametrize("n,out,k,experts", [(30, 100, 256, 200), (1000, 129, 320, 1024), (2, 2000, 512, 300), (5000, 300, 128, 64), (9, 70, 1000, 16)])
def test_experts_sums_that_need_no_rounding(spg, lib, n, out, k, experts):
    rng = np.random.default_rng(n + out + k)
    c = Call(spg, lib, rng, n, out, k, _starts(rng, n, experts, 0.5), exact=True)
    assert np.array_equal(c.rows(6, 2), c.want(6)[0])


@pytest.mark.parametrize("n,out,k,experts", [(4, 200, 8192, 3), (70, 4000, 300, 20), (3000, 1000, 384, 2), (200, 64, 64, 1000)])
def test_groups_without_any_rows(spg, lib, n, out, k, experts):
    """No row belongs to a group, or one alone: the last, a middle one, to the last layer or a middle one."""
    for first, e in ((None, 0), (n - 1, experts - 1), (n // 2, experts // 2), (0, 0)):
        starts = [n if first is None else first] * (experts + 1) if first is None else [first] * (e + 1) + [first + 1] * (experts - e)
        c = Call(spg, lib, np.random.default_rng(n), n, out, k, starts, exact=True, bias=False)
        got = c.rows(6, 2)
        assert np.array_equal(got, c.want(6)[0]) and (got == -3).all(1).sum() == (n if first is None else n - 1)


def test_starts_that_fall_or_leave_the_rows(spg, lib):
    """A start below zero or an earlier one counts as the largest before it, one beyond the last row as that."""
    for starts in ([-5, 3, 2, 9, 8, 40], [2 ** 31 - 1, 0, 5, 7], [-2 ** 31, 4, -1, 2 ** 31 - 1], [20, 10, 5, 0]):
        c = Call(spg, lib, np.random.default_rng(5), 20, 150, 260, starts, exact=True)
        assert np.array_equal(c.rows(6, 2), c.want(6)[0]), starts


@pytest.mark.parametrize("n,out,k,starts", [(1, 1, 128, None), (5, 17, 64, None), (16, 128, 300, None), (70, 777, 256, None), (300, 1000, 512, None), (2500, 2700, 128, None), (90, 130, 4096, None),
                                            (300, 1000, 256, [0, 3, 3, 200, 300]), (40, 200, 2048, [5, 10, 10, 33]), (3000, 640, 384, [0, 1, 1300, 2990])])
def test_next_operand(spg, lib, n, out, k, starts):
    """The next layer's operand is the quantised fp32 output, byte for byte, with the rows written beside it or not; what no group has is as it was."""
    import torch
    c = Call(spg, lib, np.random.default_rng(n + out + k), n, out, k, starts)
    y = torch.full((n, out), float("nan"), device="cuda")
    a, b, ref = Packed(spg, n, out, more=16), Packed(spg, n, out), Packed(spg, n, out)
    act = 3 if n % 2 else 4
    c.run(act, y, 2, out, a)
    c.run(act, None, 0, 0, b)
    none = np.ones(n, bool)
    for lo, hi in c.groups:
        none[lo:hi] = False
    y[torch.from_numpy(none).cuda()] = 0
    assert lib.spgk_fp8_quantize(y.data_ptr(), 2, out, n, None, ref.ref, None) == 0
    torch.cuda.synchronize()
    want_code, want_scale = ref.host()
    for m in (a, b):
        code, scale = m.host()
        assert np.array_equal(code[~none], want_code[~none]) and np.array_equal(scale[~none], want_scale[~none])
        assert (code[none] == 0xA5).all() and (scale[none] == 0xFF).all()
        codes, words = m.codes.cpu().numpy(), m.words.cpu().numpy()
        assert (codes[n] == 0xA5).all() and (words[-16:] == 0xFF).all() and (codes[:, -(-out // 16) * 16:] == 0xA5).all()


def test_the_longest_sums(spg, lib):
    """2^27 inputs, a thousand of them not zero: exact."""
    import torch
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("less than 8 GB free")
    rng = np.random.default_rng(2)
    k, out, n = 1 << 27, 5, 2
    w, x = Packed(spg, out, k), Packed(spg, n, k)
    for m in (w, x):
        m.codes.zero_()
        m.words[:-16] = 127
    at = np.sort(rng.choice(k, 1000, replace=False))
    at[:3], at[-1] = (0, 1, 127), k - 1
    pick = np.flatnonzero((plain.SIZES[:127] <= 8) & (plain.SIZES[:127] * 4 % 1 == 0))
    cw, cx = rng.choice(pick, (out, 1000)).astype(np.uint8), rng.choice(pick, (n, 1000)).astype(np.uint8)
    places = torch.from_numpy(at).cuda()
    w.codes[:out, places], x.codes[:n, places] = torch.from_numpy(cw).cuda(), torch.from_numpy(cx).cuda()
    y, status = torch.zeros(n, out, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_fp8(w.ref, None, 6, x.ref, y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0, lib.spgk_error_string()
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    assert np.array_equal(y.double().cpu().numpy(), plain.SIZES[cx] @ plain.SIZES[cw].T)


def test_blocks_of_nan(spg, lib):
    """A NaN block of an input makes its row NaN, one of the weights its unit; the next operand's block with them is NaN."""
    import torch
    rng = np.random.default_rng(3)
    n, out, k = 40, 300, 700
    code_w, code_x = rng.integers(0, 120, (out, k)).astype(np.uint8), rng.integers(0, 120, (n, k)).astype(np.uint8)
    scale_w, scale_x = np.full((out, 6), 120, np.uint8), np.full((n, 6), 120, np.uint8)
    scale_w[7, 5] = scale_x[9, 2] = 255
    code_x[11, 3] = 0x7F                                          # a NaN element
    w, x = Packed(spg, out, k, code_w, scale_w), Packed(spg, n, k, code_x, scale_x)
    y, nxt = torch.zeros(n, out, device="cuda"), Packed(spg, n, out)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_fp8(w.ref, None, 6, x.ref, y.data_ptr(), 2, out, nxt.ref, status.data_ptr(), None) == 0
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    nan = y.isnan().cpu().numpy()
    want = np.zeros((n, out), bool)
    want[:, 7] = want[9] = want[11] = True
    assert np.array_equal(nan, want)
    scale = nxt.host()[1]
    assert (scale[:, 0] == 255).all() and (scale[[9, 11]] == 255).all() and (np.delete(scale, [9, 11], 0)[:, 1:] < 255).all()


@pytest.mark.parametrize("low,high", [(0, 3), (250, 254), (0, 254)])
def test_scales_at_the_ends_of_their_range(spg, lib, low, high):
    """Products far below and far beyond fp32: zero or infinite where they are, else as in 64 bits."""
    import torch
    rng = np.random.default_rng(low + high)
    n, out, k = 20, 150, 128
    code_w, code_x = rng.integers(1, 126, (out, k)).astype(np.uint8), rng.integers(1, 126, (n, k)).astype(np.uint8)
    scale_w, scale_x = rng.integers(low, high + 1, (out, 1)).astype(np.uint8), rng.integers(low, high + 1, (n, 1)).astype(np.uint8)
    w, x = Packed(spg, out, k, code_w, scale_w), Packed(spg, n, k, code_x, scale_x)
    y = torch.zeros(n, out, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_fp8(w.ref, None, 6, x.ref, y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    got = y.double().cpu().numpy()
    sums = (plain.SIZES[code_x] @ plain.SIZES[code_w].T)          # all positive; then one power of two
    want = sums * np.exp2(scale_x.astype(float) - 127) * np.exp2(scale_w[:, 0].astype(float) - 127)
    huge, tiny = want > 2.0 ** 128, want < 2.0 ** -100
    assert np.isinf(got[huge]).all() and (got[tiny] <= 2.0 ** -99).all()
    rest = ~(want > 2.0 ** 127) & ~tiny
    assert (np.abs(got[rest] - want[rest]) <= want[rest] * 5 * 33 * 2.0 ** -24).all()


def test_on_another_stream_and_replayed(spg, lib):
    """Two captured graphs of the same calls on two streams, each with outputs and a status word of its own, replayed over changed inputs."""
    import torch
    rng = np.random.default_rng(1)
    c = Call(spg, lib, rng, 70, 300, 513, [0, 10, 11, 70], exact=True)
    other, other_v = _random(spg, 70, 513, rng, True)
    graphs = []
    for _ in range(2):
        stream, y, status = torch.cuda.Stream(), torch.zeros(70, 300, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert lib.spgk_experts_fp8(c.w.ref, 3, c.bd.data_ptr(), 1, c.x.ref, c.starts.data_ptr(), y.data_ptr(), 2, 300, None, status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        graphs.append((graph, stream, y, status))
    want = c.want(1)[0]
    for turn in range(2):
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, y, status in graphs:
            assert np.array_equal(y.double().cpu().numpy(), want) and status.item() == 0
        c.x.codes[:70, :513] = other.codes[:70, :513]             # the same memory, other rows
        c.x.words.copy_(other.words)
        c.xv = other_v
        c.starts.copy_(torch.tensor([0, 30, 30, 69], dtype=torch.int32))
        c.groups = plain.ranges([0, 30, 30, 69], 70)
        want = np.where(c.want(1)[0] == -3, want, c.want(1)[0])


def test_starts_that_the_launch_in_front_writes(spg, lib):
    """Starts and rows written by the launch directly in front, other ones every time, without a wait in between: none of what a layer looked at ahead is used."""
    import torch
    rng = np.random.default_rng(6)
    for n, out, k, experts in ((48, 300, 2048, 5), (900, 700, 256, 9), (5, 4000, 1024, 4)):
        c = Call(spg, lib, rng, n, out, k, [0] * experts + [n], exact=True)
        tables = [np.concatenate(([0], np.sort(rng.integers(0, n + 1, experts - 1)), [n])) for _ in range(12)]
        sources = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in tables]
        outs = [torch.zeros(n, out, device="cuda") for _ in tables]
        torch.cuda.synchronize()
        for src, y in zip(sources, outs):
            c.starts.copy_(src)
            assert lib.spgk_experts_fp8(c.w.ref, experts, c.bd.data_ptr(), 6, c.x.ref, c.starts.data_ptr(), y.data_ptr(), 2, out, None, c.status.data_ptr(), None) == 0
        assert lib.spgk_gemm_tc_status(c.status.data_ptr(), None) == 0
        for t, y in zip(tables, outs):
            c.groups = plain.ranges(t, n)
            assert np.array_equal(y.double().cpu().numpy(), c.want(6)[0])


def test_calls_at_once(spg, lib):
    """Layers of all arrangements on three streams at a time, each with outputs and a status word of its own, some of them on few SMs, in clusters and in pairs."""
    import torch
    rng = np.random.default_rng(12)
    calls = [Call(spg, lib, rng, *shape, exact=True) for shape in ((3, 300, 4096), (1, 1000, 2048), (200, 500, 1024), (700, 1500, 320), (40, 90, 3001), (64, 2100, 640))]
    calls += [Call(spg, lib, rng, 300, 400, 512, _starts(rng, 300, 9), exact=True), Call(spg, lib, rng, 2000, 600, 256, _starts(rng, 2000, 4), exact=True)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.zeros(c.n, c.out, device="cuda") for _ in streams] for c in calls]
    status = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for turn in range(6):
        for i, stream in enumerate(streams):
            for j in range(len(calls)):
                k = (j * 3 + i * 2 + turn) % len(calls)
                c, y, st = calls[k], outs[k][i].data_ptr(), stream.cuda_stream
                if c.starts is None:
                    rc = lib.spgk_layer_fp8(c.w.ref, c.bd.data_ptr(), 6, c.x.ref, y, 2, c.out, None, status[i].data_ptr(), st)
                else:
                    rc = lib.spgk_experts_fp8(c.w.ref, c.experts, c.bd.data_ptr(), 6, c.x.ref, c.starts.data_ptr(), y, 2, c.out, None, status[i].data_ptr(), st)
                assert rc == 0
    torch.cuda.synchronize()
    assert all(s.item() == 0 for s in status)
    for c, ys in zip(calls, outs):
        want = c.want(6)[0]
        for y in ys:
            assert np.array_equal(y.double().cpu().numpy(), want)


FIRST = """
import ctypes, sys, torch
sys.path.insert(0, {root!r})
import spingalett_b200 as spg
lib = spg.lib()
n, experts, top, k = 300, 6, 2, 512
x, logits = torch.randn(n, k, device="cuda"), torch.randn(n, experts, device="cuda")
def ints(m): return torch.zeros(m, dtype=torch.int32, device="cuda")
chosen, gates, starts, order, places, status = ints(n * top), torch.zeros(n * top, device="cuda"), ints(experts + 1), ints(n * top), ints(n * top), ints(1)
def matrix(rows, cols):
    m = (torch.zeros(rows, cols, dtype=torch.uint8, device="cuda"), torch.zeros(rows * 4 * (-(-cols // 512)), dtype=torch.uint8, device="cuda"))
    return m, ctypes.byref(spg.abi.Fp8(m[0].data_ptr(), m[1].data_ptr(), rows, cols, cols))
(wm, w), (xm, x8) = matrix(experts * 128, k), matrix(n * top, k)
wv = torch.randn(experts * 128, k, device="cuda")
y, out = torch.zeros(n * top, 128, device="cuda"), torch.zeros(n, 128, device="cuda")
def way():
    st = torch.cuda.current_stream().cuda_stream
    for call, args in ((lib.spgk_fp8_quantize, (wv.data_ptr(), 2, k, experts * 128, None, w)),
                       (lib.spgk_route_rows, (logits.data_ptr(), 2, experts, n, experts, top, 1, chosen.data_ptr(), gates.data_ptr(), starts.data_ptr(), order.data_ptr(), places.data_ptr())),
                       (lib.spgk_fp8_quantize, (x.data_ptr(), 2, k, n, order.data_ptr(), x8)),
                       (lib.spgk_experts_fp8, (w, experts, None, 1, x8, starts.data_ptr(), y.data_ptr(), 2, 128, None, status.data_ptr())),
                       (lib.spgk_combine_rows, (y.data_ptr(), 2, 128, n * top, places.data_ptr(), gates.data_ptr(), n, top, 128, out.data_ptr(), 2, 128))):
        assert call(*args, st) == 0, lib.spgk_error_string()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    way()
graph.replay()
torch.cuda.synchronize()
got = out.clone()
out.zero_()
way()
torch.cuda.synchronize()
assert status.item() == 0 and torch.equal(got, out) and got.abs().max() > 1
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture(lib):
    import subprocess
    import sys
    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=ROOT)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_offsets_beyond_32_bits(spg, lib):
    """Weights of 5 GB of which the last layer is used, rows of the output and of what is quantised 4 GB apart."""
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("less than 40 GB free")
    rng = np.random.default_rng(8)
    experts, out, k, n = 610, 1024, 8192, 5
    w = Packed(spg, experts * out, k)
    code = rng.choice(np.flatnonzero((plain.SIZES[:127] <= 8) & (plain.SIZES[:127] * 4 % 1 == 0)), (out, k)).astype(np.uint8)
    w.codes[(experts - 1) * out:experts * out] = torch.from_numpy(code).cuda()
    words = w.words[:-16].view(-1, experts * out, 4)
    words.fill_(127)
    assert w.codes.numel() > 2 ** 32 and w.codes[-1:].data_ptr() - w.codes.data_ptr() > 2 ** 32
    x, xv = _random(spg, n, k, rng, True)
    starts = torch.full((experts + 1,), 2, dtype=torch.int32, device="cuda")
    starts[0], starts[-1] = 0, n                                   # two rows to the first layer, the rest to the last
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ldy = 1 << 30
    y = torch.zeros((n - 1) * ldy + out, dtype=torch.float16, device="cuda")
    assert lib.spgk_experts_fp8(w.ref, experts, None, 6, x.ref, starts.data_ptr(), y.data_ptr(), 0, ldy, None, status.data_ptr(), None) == 0, lib.spgk_error_string()
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    want = (torch.from_numpy(xv[2:]) @ torch.from_numpy(plain.SIZES[code]).T).to(torch.float16)
    got = torch.stack([y[r * ldy:r * ldy + out] for r in range(2, n)]).cpu()
    assert torch.equal(got, want)
    # the same rows quantised from where they lie, taken by index, and added up
    index = torch.tensor([4, 2], dtype=torch.int32, device="cuda")
    m = Packed(spg, 2, out)
    assert lib.spgk_fp8_quantize(y.data_ptr(), 0, ldy, n, index.data_ptr(), m.ref, None) == 0
    torch.cuda.synchronize()
    code_w, scale_w = plain.quantize(got.double().numpy()[[2, 0]])
    code, scale = m.host()
    assert np.array_equal(code, code_w) and np.array_equal(scale, scale_w)
    places, gates = torch.tensor([[3, 4]], dtype=torch.int32, device="cuda"), torch.tensor([[0.5, 0.25]], device="cuda")
    total = torch.zeros(out, device="cuda")
    assert lib.spgk_combine_rows(y.data_ptr(), 0, ldy, n, places.data_ptr(), gates.data_ptr(), 1, 2, out, total.data_ptr(), 2, out, None) == 0
    assert torch.allclose(total.cpu(), 0.5 * got[1].float() + 0.25 * got[2].float(), rtol=2.0 ** -22, atol=0)


def test_operands_that_are_views(spg, lib):
    """Rows taken out of a larger matrix, from any row on: its own codes and the scales' pitch, in a matrix of their own made by an index."""
    import torch
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((50, 900)).astype(np.float32)).cuda()
    part = x[7:40, 100:877]                                        # neither its first row nor its column lies on 16 bytes
    m = Packed(spg, 33, 777)
    assert lib.spgk_fp8_quantize(part.data_ptr(), 2, x.stride(0), 33, None, m.ref, None) == 0
    torch.cuda.synchronize()
    code_w, scale_w = plain.quantize(part.double().cpu().numpy())
    code, scale = m.host()
    assert np.array_equal(code, code_w) and np.array_equal(scale, scale_w)
    w, wv = _random(spg, 70, 777, rng)
    y = torch.full((40, 80), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    into = y[3:36, 5:75]
    assert lib.spgk_layer_fp8(w.ref, None, 6, m.ref, into.data_ptr(), 2, 80, None, status.data_ptr(), None) == 0
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    want = plain.values(code_w, scale_w) @ wv.T
    size = np.abs(plain.values(code_w, scale_w)) @ np.abs(wv).T
    assert (np.abs(into.double().cpu().numpy() - want) <= size * 26 * 33 * 2.0 ** -24).all()
    into.fill_(5.0)
    assert (y == 5).all()                                          # nothing beside it was written
