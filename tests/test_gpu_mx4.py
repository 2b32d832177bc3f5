"""Microscaled 4-bit numbers on the GPU: quantising and back byte for byte, the layer against sums in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import mx4_plain as plain

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
    """A matrix on the device, with what it points to."""

    def __init__(self, spg, rows, cols, codes=None, tiles=None, more=0):
        import torch
        self.rows, self.cols, self.pitch = rows, cols, -(-cols // 32) * 16 + more
        self.codes = torch.full((rows + 1, self.pitch), 0xA5, dtype=torch.uint8, device="cuda")
        self.tiles = torch.full((-(-rows // 128) * -(-cols // 128) * 512 + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        if codes is not None:
            self.codes[:rows] = torch.from_numpy(codes).cuda()
            self.tiles[:-16] = torch.from_numpy(tiles).cuda()
        self.m = spg.abi.Mx4(self.codes.data_ptr(), self.tiles.data_ptr(), rows, cols, self.pitch)
        self.ref = C.byref(self.m)

    def host(self):
        return plain.unpack(self.codes.cpu().numpy(), self.tiles.cpu().numpy(), self.rows, self.cols)


def _random(spg, rows, cols, rng, exact=False, more=0):
    """Random codes and scales; exact: scales close enough for sums without rounding."""
    code = rng.integers(0, 16, (rows, -(-cols // 32) * 32)).astype(np.uint8)
    code[:, cols:] = 0
    scale = rng.integers(126, 129, (rows, code.shape[1] // 32)) if exact else rng.integers(115, 134, (rows, code.shape[1] // 32))
    scale = scale.astype(np.uint8)
    codes, tiles = plain.pack(code, scale, cols, -(-cols // 32) * 16 + more)
    return Packed(spg, rows, cols, codes, tiles, more), plain.values(code, scale, cols)


def _values_with_extremes(rows, cols, t, rng):
    import torch
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    flat = x.reshape(-1)
    n = flat.size
    flat[:: 37] = 0.0
    if rows > 2:
        x[1] = 0.0                                           # a row of zeros
        x[2, : cols // 2] *= 2.0 ** -140                     # far below the smallest scale
    if rows > 5:
        x[3] = np.resize([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0], cols)   # half way
        x[4, :: 3] = -0.0
        x[5, cols // 2] = np.nan
    if rows > 7:
        x[6, 0] = np.inf
        x[7, cols - 1] = -np.inf
    if rows > 8 and t != 0:
        x[8] = np.resize([3.3e38, -1e38, 1e-44, 2.0 ** -126, 3.0 * 2.0 ** -127], cols)
    assert n
    return torch.from_numpy(x.astype(np.float32)).to(_dtype(t))


@pytest.mark.parametrize("t", [2, 1, 0])
@pytest.mark.parametrize("rows,cols,pad,off", [(1, 1, 0, 0), (1, 8192, 0, 0), (9, 31, 0, 0), (9, 32, 0, 0), (10, 33, 3, 0), (130, 777, 24, 0), (257, 129, 1, 1), (12, 1000, 0, 3), (300, 256, 8, 8), (64, 4100, 4, 0)])
def test_quantize_and_back(spg, lib, t, rows, cols, pad, off):
    import torch
    rng = np.random.default_rng(rows * 1000 + cols + t)
    x = _values_with_extremes(rows, cols, t, rng)
    buf = torch.zeros(rows * (cols + pad) + off, dtype=x.dtype, device="cuda")
    view = buf[off:].view(rows, cols + pad)
    view[:, :cols] = x.cuda()
    view[:, cols:] = float("nan")                             # what is beside a row is not read
    m = Packed(spg, rows, cols, more=16 if pad else 0)
    assert lib.spgk_mx4_quantize(view.data_ptr(), t, cols + pad, m.ref, None) == 0, lib.spgk_error_string()
    torch.cuda.synchronize()
    want_code, want_scale = plain.quantize(x.double().numpy())
    code, scale = m.host()
    assert np.array_equal(scale, want_scale)
    assert np.array_equal(code, want_code)
    codes, tiles = m.codes.cpu().numpy(), m.tiles.cpu().numpy()
    assert (codes[rows] == 0xA5).all() and (tiles[-16:] == 0xFF).all() and (codes[:, -(-cols // 32) * 16:] == 0xA5).all()
    used = np.zeros(tiles.size - 16, bool)
    r, b = np.meshgrid(np.arange(rows), np.arange(scale.shape[1]), indexing="ij")
    used[plain.scale_place(cols, r, b)] = True
    assert (tiles[:-16][~used] == 0).all()                    # tiles are whole
    want = plain.values(want_code, want_scale, cols)
    for to in (2, 1, 0):
        y = torch.full((rows + 1, cols + pad), 7.0, dtype=_dtype(to), device="cuda")
        assert lib.spgk_mx4_dequantize(m.ref, y.data_ptr(), to, cols + pad, None) == 0, lib.spgk_error_string()
        got = y.cpu()
        assert (got[rows] == 7).all() and (got[:, cols:] == 7).all()
        expect = torch.from_numpy(want).float().to(_dtype(to))
        assert torch.equal(torch.nan_to_num(got[:rows, :cols], 12345.0), torch.nan_to_num(expect, 12345.0))
        assert torch.equal(torch.isnan(got[:rows, :cols]), torch.isnan(expect))


SHAPES = [(1, 1, 1), (1, 10, 1000), (2, 333, 777), (16, 128, 256), (17, 129, 31), (33, 300, 64), (65, 257, 1025), (128, 512, 784), (300, 1000, 512), (513, 130, 4100), (600, 64, 33),
          (1, 128, 16384), (8, 200, 8192), (40, 96, 3001), (700, 1500, 320), (129, 1, 200), (257, 2, 40), (2500, 2700, 300), (4100, 1100, 70), (90, 33, 20000),
          (9, 900, 2048), (24, 130, 4096), (64, 1030, 4096), (100, 260, 2048), (128, 1100, 1024), (300, 390, 4096)]     # tiles that two to eight CTAs share


def _layer(spg, lib, rng, n, out, k, act, t, exact, bias=True):
    import torch
    w, wv = _random(spg, out, k, rng, exact)
    x, xv = _random(spg, n, k, rng, exact, more=32 if n % 2 else 0)
    b = (rng.integers(-8, 9, out) if exact else rng.standard_normal(out)).astype(np.float32)
    bd = torch.from_numpy(b).cuda()
    ldy = out + n % 3
    y = torch.full((n + 1, ldy), -3.0, dtype=_dtype(t), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_mx4(w.ref, bd.data_ptr() if bias else None, act, x.ref, y.data_ptr(), t, ldy, None, status.data_ptr(), None) == 0, lib.spgk_error_string()
    lib.spgk_gemm_tc_status.argtypes = [C.c_void_p, C.c_void_p]
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0, lib.spgk_error_string()
    got = y.double().cpu().numpy()
    assert (got[n] == -3).all() and (got[:, out:] == -3).all()
    with np.errstate(over="ignore"):
        want = plain.ACTS[act](xv @ wv.T + (b if bias else 0))
    return got[:n, :out], want, np.abs(xv) @ np.abs(wv).T + np.abs(b), (w, x, bd, wv, xv)


@pytest.mark.parametrize("n,out,k", [s for s in SHAPES if s[2] <= 4100])      # (longer sums would need more bits)
def test_layer_sums_that_need_no_rounding(spg, lib, n, out, k):
    """Whole multiples of 1/16 below 2^19: every sum is exact in 32 bits, whatever its order."""
    got, want, *_ = _layer(spg, lib, np.random.default_rng(n + out + k), n, out, k, 6, 2, True)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("n,out,k", SHAPES)
@pytest.mark.parametrize("t", [2, 1, 0])
def test_layer_against_64_bits(spg, lib, n, out, k, t):
    act = (n + out + k + t) % 7
    got, want, size, _ = _layer(spg, lib, np.random.default_rng(n * 3 + out + k), n, out, k, act, t, False, bias=(n + t) % 4 != 0)
    # A step adds 64 products to the sum: 65 numbers, of which each may lose what lies below 2^-24 of the largest, itself no larger than the sum of
    # all magnitudes; then the bias, the activation (no steeper than 1; 4 ulp of its own functions) and the rounding of the output.
    steps = -(-k // 64) + 1
    tol = steps * 65 * 2.0 ** -24 * size + np.abs(want) * (HALF[t] + 4 * 2.0 ** -23) + (2.0 ** -25 if t == 0 else 0)
    big = np.abs(want) > 65504
    if t == 0:
        assert (np.isinf(got) | (np.abs(got) > 65000))[big].all()
        got, want, tol = got[~big], want[~big], tol[~big]
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("n,out,k", [s for s in SHAPES if s[0] * s[1] > 1])
def test_layer_output_as_the_next_operand(spg, lib, n, out, k):
    """Quantised in the epilogue: byte for byte what spgk_mx4_quantize makes of the fp32 output."""
    import torch
    act = (n + out + k) % 5
    rng = np.random.default_rng(n + 5 * out + k)
    got, want, size, (w, x, b, _, _) = _layer(spg, lib, rng, n, out, k, act, 2, False)
    y = torch.full((n, out), -3.0, dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, c, both = Packed(spg, n, out), Packed(spg, n, out, more=16), Packed(spg, n, out)
    assert lib.spgk_layer_mx4(w.ref, b.data_ptr(), act, x.ref, None, 0, 0, a.ref, status.data_ptr(), None) == 0, lib.spgk_error_string()
    assert lib.spgk_layer_mx4(w.ref, b.data_ptr(), act, x.ref, y.data_ptr(), 2, out, c.ref, status.data_ptr(), None) == 0, lib.spgk_error_string()
    assert np.array_equal(y.double().cpu().numpy(), got)
    assert lib.spgk_mx4_quantize(y.data_ptr(), 2, out, both.ref, None) == 0
    for m in (a, c):
        for mine, theirs in zip(m.host(), both.host()):
            assert np.array_equal(mine, theirs)
        assert (m.codes[n].cpu().numpy() == 0xA5).all() and (m.tiles[-16:].cpu().numpy() == 0xFF).all()
    # and it is an operand: the scales of blocks beyond the matrix are no NaN
    got2 = torch.empty((n, out), dtype=torch.float32, device="cuda")
    unit, uv = _random(spg, out, out, rng, True)
    assert lib.spgk_layer_mx4(unit.ref, None, 6, a.ref, got2.data_ptr(), 2, out, None, status.data_ptr(), None) == 0
    assert np.isfinite(got2.cpu().numpy()).all()
    xv = plain.values(*a.host(), out)
    steps = -(-out // 64) + 1
    assert (np.abs(got2.double().cpu().numpy() - xv @ uv.T) <= steps * 65 * 2.0 ** -24 * (np.abs(xv) @ np.abs(uv).T) + 1e-30).all()


@pytest.mark.parametrize("ws,xs", [(254, 0), (0, 254), (253, 3), (20, 240), (127, 127)])
@pytest.mark.parametrize("n", [3, 100, 600])
def test_scales_at_their_ends(spg, lib, ws, xs, n):
    """Scales at the ends of their range whose products are near one: sums that need no rounding, and values in the range of fp32."""
    import torch
    rng = np.random.default_rng(ws + n)
    out, k = 150, 160
    half = 2.0 ** (ws + xs - 254)
    mats = []
    for rows, byte in ((out, ws), (n, xs)):
        code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
        scale = np.full((rows, k // 32), byte, np.uint8)
        mats.append((Packed(spg, rows, k, *plain.pack(code, scale, k)), plain.values(code, np.full_like(scale, 127), k)))
    y = torch.empty((n, out), dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_mx4(mats[0][0].ref, None, 6, mats[1][0].ref, y.data_ptr(), 2, out, None, status.data_ptr(), None) == 0
    assert np.array_equal(y.double().cpu().numpy(), mats[1][1] @ mats[0][1].T * half)


@pytest.mark.parametrize("n,out,k", [(5, 140, 300), (140, 300, 300), (600, 140, 700)])
def test_nan_blocks_stay_in_their_rows(spg, lib, n, out, k):
    import torch
    rng = np.random.default_rng(7)
    w, _ = _random(spg, out, k, rng)
    x, _ = _random(spg, n, k, rng)
    w.tiles[plain.scale_place(k, 3, 1)] = 255
    x.tiles[plain.scale_place(k, 2, 0)] = 255
    y = torch.zeros((n, out), dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    nxt = Packed(spg, n, out)
    assert lib.spgk_layer_mx4(w.ref, None, 6, x.ref, y.data_ptr(), 2, out, nxt.ref, status.data_ptr(), None) == 0
    bad = np.isnan(y.cpu().numpy())
    want = np.zeros_like(bad)
    want[2], want[:, 3] = True, True
    assert np.array_equal(bad, want)
    scale = nxt.host()[1]
    assert (scale[2] == 255).all() and (scale[:, 0] == 255).all() and (np.delete(scale, 2, 0)[:, 1:] != 255).all()


def test_streams_replay_and_two_calls_at_once(spg, lib):
    """Two streams, then a captured sequence replayed on new inputs: the results of plain calls."""
    import torch
    rng = np.random.default_rng(3)
    w, wv = _random(spg, 500, 900, rng)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    xs = [torch.randn(70, 900, device="cuda") for _ in range(2)]
    packed = [Packed(spg, 70, 900) for _ in range(2)]
    ys = [torch.zeros(70, 500, device="cuda") for _ in range(2)]
    status = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()

    def go(i, stream):
        assert lib.spgk_mx4_quantize(xs[i].data_ptr(), 2, 900, packed[i].ref, stream) == 0
        assert lib.spgk_layer_mx4(w.ref, None, 1, packed[i].ref, ys[i].data_ptr(), 2, 500, None, status[i].data_ptr(), stream) == 0

    def check(i):
        x = plain.values(*plain.quantize(xs[i].double().cpu().numpy()), 900)
        tol = 16 * 65 * 2.0 ** -24 * (np.abs(x) @ np.abs(wv).T) + 1e-6
        assert (np.abs(ys[i].double().cpu().numpy() - np.maximum(x @ wv.T, 0)) <= tol).all()
    for _ in range(3):
        for i in range(2):
            go(i, sides[i].cuda_stream)
    torch.cuda.synchronize()
    check(0)
    check(1)
    go(0, sides[0].cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=sides[0]):
        go(0, sides[0].cuda_stream)
    xs[0].normal_()
    ys[0].zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    check(0)
    del graph


def test_a_served_forward(spg, lib):
    """Rows quantised, a hidden layer that stays in 4 bits, logits, a token a row: every step against its plain form on what the step before gave."""
    import torch
    rng = np.random.default_rng(11)
    n, k, hidden, classes = 37, 784, 1000, 10007
    w1, _ = _random(spg, hidden, k, rng)
    w2, w2v = _random(spg, classes, hidden, rng)
    b1, b2 = torch.randn(hidden, device="cuda"), torch.randn(classes, device="cuda")
    x = torch.rand(n, k, device="cuda")
    x4, h4 = Packed(spg, n, k), Packed(spg, n, hidden)
    logits = torch.empty((n, classes), dtype=torch.float32, device="cuda")
    t, p, u = torch.full((n,), 40.0, device="cuda"), torch.full((n,), 0.9, device="cuda"), torch.rand(n, device="cuda")
    tokens, status = torch.empty(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    s = side.cuda_stream
    assert lib.spgk_mx4_quantize(x.data_ptr(), 2, k, x4.ref, s) == 0
    assert lib.spgk_layer_mx4(w1.ref, b1.data_ptr(), 4, x4.ref, None, 0, 0, h4.ref, status.data_ptr(), s) == 0
    assert lib.spgk_layer_mx4(w2.ref, b2.data_ptr(), 6, h4.ref, logits.data_ptr(), 2, classes, None, status.data_ptr(), s) == 0
    assert lib.spgk_sample_rows(logits.data_ptr(), 2, classes, n, classes, t.data_ptr(), None, p.data_ptr(), None, u.data_ptr(), tokens.data_ptr(), None, None, s) == 0
    torch.cuda.synchronize()
    assert status.item() == 0
    hv = plain.values(*h4.host(), hidden)
    want = hv @ w2v.T + b2.double().cpu().numpy()
    got = logits.double().cpu().numpy()
    assert (np.abs(got - want) <= 17 * 65 * 2.0 ** -24 * (np.abs(hv) @ np.abs(w2v).T + 5)).all()
    assert tokens.cpu().tolist() == [plain.sample_row(got[i], 40.0, None, float(np.float32(0.9)), None, u[i].item())[0] for i in range(n)]
