"""Microscaled 4-bit numbers at sizes that take the other ways: layers on pairs of CTAs with several tiles and long rings, quantising in wider shares of a tile."""
import ctypes as C

import numpy as np
import pytest

import mx4_plain as plain
from test_gpu_mx4 import HALF, Packed, _dtype, _random, _values_with_extremes, lib  # noqa: F401  (lib: fixture)

pytestmark = pytest.mark.gpu

# More than 74 tiles of 256 x 256, so that pairs have two to four each; more than six k-blocks of 256, with 1, 64, 100, 192 and 254 inputs in the last one; a single one; many
PAIRS = [(3001, 5003, 1537), (2999, 5100, 1600), (3001, 5003, 1636), (5003, 2900, 1728), (3001, 5003, 1790), (300, 30000, 1801), (4100, 4100, 70), (2500, 2700, 20000)]


def _matrix(spg, rows, cols, rng, byte):
    """Random codes with one scale."""
    code = rng.integers(0, 16, (rows, -(-cols // 32) * 32)).astype(np.uint8)
    code[:, cols:] = 0
    scale = np.full((rows, code.shape[1] // 32), byte, np.uint8)
    return Packed(spg, rows, cols, *plain.pack(code, scale, cols)), plain.values(code, np.full_like(scale, 127), cols)


def _product(xv, wv):
    import torch
    return torch.from_numpy(xv).cuda() @ torch.from_numpy(wv).cuda().T


def _run(lib, w, x, bias, act, y, t, nxt=None):
    import torch
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_layer_mx4(w.ref, None if bias is None else bias.data_ptr(), act, x.ref, y.data_ptr(), t, y.stride(0), None if nxt is None else nxt.ref, status.data_ptr(), None) == 0, lib.spgk_error_string()
    return lib.spgk_gemm_tc_status(status.data_ptr(), None)


def _is_of_pairs(lib, w, x, y):
    """Where pairs of CTAs have the tiles, giving up leaves only the last one of each alone; single CTAs have one each."""
    y.fill_(float("nan"))
    lib.spgk_selftest_impatient(1)
    try:
        assert _run(lib, w, x, None, 6, y, 2) == -4
    finally:
        lib.spgk_selftest_impatient(0)
    return bool(y.isfinite().any())


@pytest.mark.parametrize("n,out,k", PAIRS)
def test_sums_that_need_no_rounding_in_pairs(spg, lib, n, out, k):
    """Products are whole multiples of 1/4 up to 36, so every sum is exact in 32 bits, and a lost or doubled step of 64 inputs shows.  Rows of each type, and the next operand."""
    import torch
    rng = np.random.default_rng(n + out + k)
    (w, wv), (x, xv) = _matrix(spg, out, k, rng, 127), _matrix(spg, n, k, rng, 127)
    bias = torch.from_numpy(rng.integers(-8, 9, out).astype(np.float32)).cuda()
    want = _product(xv, wv) + bias.double()
    assert _is_of_pairs(lib, w, x, torch.empty((n, out), device="cuda"))
    for t in (2, 1, 0):
        ld = out + 3 * (t == 1)
        y = torch.full((n + 1, ld), -3.0, dtype=_dtype(t), device="cuda")
        nxt = Packed(spg, n, out, more=16 * (t == 0))
        assert _run(lib, w, x, bias, 6, y[:n], t, nxt) == 0, lib.spgk_error_string()
        assert torch.equal(y[:n, :out], want.to(_dtype(t)))
        assert (y[n] == -3).all() and (y[:, out:] == -3).all()
        assert (nxt.codes[n] == 0xA5).all() and (nxt.tiles[-16:] == 0xFF).all()
        theirs = Packed(spg, n, out)
        exact = want.float()
        assert lib.spgk_mx4_quantize(exact.data_ptr(), 2, out, theirs.ref, None) == 0
        for mine, their in zip(nxt.host(), theirs.host()):
            assert np.array_equal(mine, their)


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
def test_activations_and_scales_in_pairs(spg, lib, act):
    import torch
    n, out, k = 3001, 5003, 1636
    rng = np.random.default_rng(act)
    (w, wv), (x, xv) = _random(spg, out, k, rng), _random(spg, n, k, rng)
    b = rng.standard_normal(out).astype(np.float32)
    bias, t = torch.from_numpy(b).cuda(), act % 3
    y = torch.empty((n, out), dtype=_dtype(t), device="cuda")
    assert _is_of_pairs(lib, w, x, torch.empty((n, out), device="cuda"))
    assert _run(lib, w, x, bias, act, y, t) == 0
    with np.errstate(over="ignore"):
        want = plain.ACTS[act](_product(xv, wv).cpu().numpy() + b)
    size = _product(np.abs(xv), np.abs(wv)).cpu().numpy() + np.abs(b)
    # 65 numbers a step of 64 inputs, of which each may lose what lies below 2^-24 of the largest; the activation (no steeper than 1; 4 ulp of its own functions); the output's rounding
    tol = (-(-k // 64) + 1) * 65 * 2.0 ** -24 * size + np.abs(want) * (HALF[t] + 4 * 2.0 ** -23) + (2.0 ** -25 if t == 0 else 0)
    got = y.double().cpu().numpy()
    big = np.abs(want) > 65504
    if t == 0:
        assert (np.isinf(got) | (np.abs(got) > 65000))[big].all()
        got, want, tol = got[~big], want[~big], tol[~big]
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("ws,xs", [(254, 0), (0, 254), (253, 3), (20, 240), (127, 127)])
def test_scales_at_their_ends_in_pairs(spg, lib, ws, xs):
    import torch
    n, out, k = 2500, 2700, 1700
    rng = np.random.default_rng(ws + n)
    (w, wv), (x, xv) = _matrix(spg, out, k, rng, ws), _matrix(spg, n, k, rng, xs)
    y = torch.empty((n, out), dtype=torch.float32, device="cuda")
    assert _run(lib, w, x, None, 6, y, 2) == 0
    assert torch.equal(y.double(), _product(xv, wv) * 2.0 ** (ws + xs - 254))


def test_nan_blocks_stay_in_their_rows_in_pairs(spg, lib):
    import torch
    n, out, k = 2500, 2700, 1700
    rng = np.random.default_rng(7)
    (w, _), (x, _) = _random(spg, out, k, rng), _random(spg, n, k, rng)
    units, rows = [3, 127, 128, 300, 2699], [0, 2, 255, 256, 2499]
    for i, (u, r) in enumerate(zip(units, rows)):
        w.tiles[plain.scale_place(k, u, (13 * i) % 54)] = 255
        x.tiles[plain.scale_place(k, r, 53 - 11 * i)] = 255
    y = torch.zeros((n, out), dtype=torch.float32, device="cuda")
    nxt = Packed(spg, n, out)
    assert _run(lib, w, x, None, 6, y, 2, nxt) == 0
    want = np.zeros((n, out), bool)
    want[rows], want[:, units] = True, True
    assert np.array_equal(np.isnan(y.cpu().numpy()), want)
    blocks = np.zeros((n, -(-out // 32)), bool)
    blocks[rows], blocks[:, [u // 32 for u in units]] = True, True
    assert np.array_equal(nxt.host()[1] == 255, blocks)


def _quantize(x):
    """plain.quantize of device rows in 64 bits, some rows at a time: (codes, scales) on the device."""
    import torch
    sizes = torch.tensor(plain.SIZES, dtype=torch.float64, device="cuda")
    codes, scales = [], []
    for part in x.split(512):
        v = torch.nn.functional.pad(part.double(), (0, -part.shape[1] % 32)).view(len(part), -1, 32)
        bad = ~v.isfinite().all(-1)
        a = torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v).abs()
        e = torch.where(a.amax(-1) > 0, torch.frexp(a.amax(-1))[1] - 3, -127).clamp(min=-127)
        q = (a / torch.exp2(e.double()).unsqueeze(-1)).clamp(max=6.0)
        code = torch.zeros_like(v, dtype=torch.uint8)
        for i in range(1, 8):
            half = (sizes[i - 1] + sizes[i]) / 2
            code += (q > half) | ((q == half) if i % 2 == 0 else torch.zeros_like(q, dtype=torch.bool))
        code |= torch.signbit(v).to(torch.uint8) << 3
        codes.append(torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(1))
        scales.append(torch.where(bad, 255, e + 127).to(torch.uint8))
    return torch.cat(codes), torch.cat(scales)


@pytest.mark.parametrize("t", [2, 1, 0])
@pytest.mark.parametrize("rows,cols,pad,off", [(3001, 4001, 7, 0), (3001, 4001, 8, 1), (2990, 4100, 4, 0), (5003, 8001, 31, 0), (5003, 8001, 0, 0), (5100, 7970, 6, 3)])
def test_quantize_and_back_in_wider_shares(spg, lib, t, rows, cols, pad, off):
    """From 592 tiles of scales on a block of threads has 64 rows of a tile, from 2368 on all of them, four rows of a group of lanes at a time; rows on 16 bytes and off them."""
    import torch
    assert -(-rows // 128) * -(-cols // 128) >= (2368 if rows > 5000 else 592) and rows % 128
    rng = np.random.default_rng(rows + cols + t)
    x = _values_with_extremes(rows, cols, t, rng).cuda()
    assert np.array_equal(_quantize(x[:40])[0].cpu().numpy(), plain.quantize(x[:40].double().cpu().numpy())[0])          # (the plain form's other spelling)
    buf = torch.full((rows * (cols + pad) + off,), float("nan"), dtype=x.dtype, device="cuda")
    view = buf[off:].view(rows, cols + pad)
    view[:, :cols] = x
    m = Packed(spg, rows, cols, more=16 if pad else 0)
    assert lib.spgk_mx4_quantize(view.data_ptr(), t, cols + pad, m.ref, None) == 0, lib.spgk_error_string()
    code, scale = _quantize(x)
    blocks = -(-cols // 32)
    packed = code[:, 0::2] | code[:, 1::2] << 4
    assert torch.equal(m.codes[:rows, :blocks * 16], packed)
    assert (m.codes[rows] == 0xA5).all() and (m.tiles[-16:] == 0xFF).all() and (m.codes[:, blocks * 16:] == 0xA5).all()
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    tiles = torch.zeros(m.tiles.numel() - 16, dtype=torch.uint8, device="cuda")
    tiles[torch.from_numpy(plain.scale_place(cols, r, b)).cuda()] = scale
    assert torch.equal(m.tiles[:-16], tiles)                     # whole tiles, zeros where there is no block
    unit = torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127))
    size = torch.tensor(list(plain.SIZES) + [-s for s in plain.SIZES], dtype=torch.float64, device="cuda")
    want = (size[code.long()].view(rows, blocks, 32) * unit.unsqueeze(-1)).flatten(1)[:, :cols].float()
    for to in (2, 1, 0):
        out = torch.full(((rows + 1) * (cols + pad) + off,), 7.0, dtype=_dtype(to), device="cuda")
        y = out[off:].view(rows + 1, cols + pad)
        assert lib.spgk_mx4_dequantize(m.ref, y.data_ptr(), to, cols + pad, None) == 0, lib.spgk_error_string()
        assert (y[rows] == 7).all() and (y[:, cols:] == 7).all() and (out[:off] == 7).all()
        got, expect = y[:rows, :cols], want.to(_dtype(to))
        assert torch.equal(got.isnan(), expect.isnan()) and torch.equal(got.nan_to_num(12345.0), expect.nan_to_num(12345.0))
