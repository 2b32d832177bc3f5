"""Rows to experts and back on the GPU: choice, gates and order against a plain form, weighted sums in 64 bits, and the whole way through two layers of experts."""
import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_fp8 import HALF, Packed, _dtype, _random, lib  # noqa: F401  (lib: fixture)

pytestmark = pytest.mark.gpu


class Route:
    def __init__(self, n, experts, top):
        import torch

        def ints(count):
            return torch.full((count + 1,), -77, dtype=torch.int32, device="cuda")
        self.n, self.experts, self.top = n, experts, top
        self.chosen, self.starts, self.order, self.places = ints(n * top), ints(experts + 1), ints(n * top), ints(n * top)
        self.gates = torch.full((n * top + 1,), -77.0, device="cuda")

    def run(self, lib, x, t, ld, normalise, stream=None):
        assert lib.spgk_route_rows(x.data_ptr(), t, ld, self.n, self.experts, self.top, normalise, self.chosen.data_ptr(), self.gates.data_ptr(), self.starts.data_ptr(),
                                   self.order.data_ptr(), self.places.data_ptr(), stream) == 0, lib.spgk_error_string()

    def check(self, logits, normalise):
        chosen, gates, starts, order, places = plain.route(logits, self.top, normalise)
        got = [v.cpu().numpy() for v in (self.chosen, self.gates, self.starts, self.order, self.places)]
        assert all(v[-1] == -77 for v in got)
        assert np.array_equal(got[0][:-1].reshape(self.n, -1) if self.n else got[0][:-1], chosen if self.n else [])
        assert np.array_equal(got[2][:-1], starts)
        assert np.array_equal(got[3][:-1], order)
        assert np.array_equal(got[4][:-1], places.reshape(-1))
        # a weight: the difference's rounding (2^-24 of it, up to 88 where the weight is not zero), 2 ulp of expf; the sum: every term's, and one rounding for each of the
        # additions a value goes through (32 of a lane, 5 across); the division's
        far = np.minimum(np.abs(np.where(np.isfinite(logits), logits, 0)).max(initial=0) * 2, 104)
        assert np.allclose(got[1][:-1], gates.reshape(-1), rtol=2 * (far + 4) * 2.0 ** -24 + 40 * 2.0 ** -24, atol=2.0 ** -126)


def _logits(rng, n, experts, kind):
    l = rng.standard_normal((n, experts)) * 2
    if kind == "ties":
        l = np.round(l)
        l[rng.random(l.shape) < 0.1] = -0.0
    if kind in ("masked", "ties"):
        l[rng.random(l.shape) < 0.4] = -np.inf
        l[rng.random(l.shape) < 0.05] = np.nan
        if n > 3:
            l[1], l[2, 1:], l[n - 1] = -np.inf, -np.inf, np.nan
            l[3, rng.integers(0, experts, 2)] = np.inf
    if kind == "lowest":
        l[:] = -3.0e38
        l[:, ::3] = -np.inf
        l[:, experts // 2] = -1e30
    if kind == "small":                                          # subnormals of 16 bits, of either sign, and both zeros
        l = rng.integers(-3, 4, (n, experts)) * 2.0 ** -24
        l[rng.random(l.shape) < 0.2] = -0.0
    if kind == "one":                                            # all rows to the same experts
        l[:] = -np.arange(experts)
    return l


@pytest.mark.parametrize("kind", ["plain", "ties", "masked", "lowest", "small", "one"])
@pytest.mark.parametrize("n,experts,top,pad,t", [(1, 1, 1, 0, 2), (1, 64, 2, 0, 2), (3, 2, 2, 0, 1), (33, 7, 3, 1, 0), (100, 32, 32, 0, 2), (257, 33, 4, 3, 1), (300, 100, 8, 0, 2), (1000, 256, 8, 8, 0), (700, 257, 5, 0, 2),
                                                 (9, 1024, 32, 0, 1), (2500, 1000, 6, 1, 2), (5000, 3, 1, 0, 2), (0, 16, 2, 0, 2)])
def test_route(lib, kind, n, experts, top, pad, t):
    import torch
    rng = np.random.default_rng(n * 7 + experts + top)
    if kind == "lowest" and t == 0:
        pytest.skip("beyond fp16")
    full = torch.full((n, experts + pad), 1e4 if pad else 0.0, dtype=_dtype(t), device="cuda")        # what is beside a row is not read
    full[:, :experts] = torch.from_numpy(_logits(rng, n, experts, kind)).to(_dtype(t)).cuda()
    logits = full[:, :experts].double().cpu().numpy()
    for normalise in (0, 1):
        r = Route(n, experts, top)
        r.run(lib, full, t, experts + pad, normalise)
        torch.cuda.synchronize()
        r.check(logits, normalise)


@pytest.mark.parametrize("n,experts,top", [(16384, 256, 8), (70001, 64, 2), (40000, 1024, 3)])
def test_long_routes(lib, n, experts, top):
    """Against a sort of all pairs: the plain form would take too long."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    x = torch.round(torch.randn(n, experts, device="cuda", generator=g) * 8) / 4
    x[torch.rand(x.shape, device="cuda", generator=g) < 0.3] = float("-inf")
    x[::1000] = float("-inf")
    r = Route(n, experts, top)
    r.run(lib, x, 2, experts, 1)
    by = torch.sort(x, dim=1, descending=True, stable=True)
    open_ = by[0][:, :top] > float("-inf")
    chosen = torch.where(open_, by[1][:, :top], -1)
    assert torch.equal(r.chosen[:-1].view(n, top).long(), chosen)
    flat = torch.where(open_, chosen, experts).view(-1)
    order = torch.sort(flat, stable=True)[1]
    total = int(open_.sum())
    starts = torch.searchsorted(flat[order], torch.arange(experts + 1, device="cuda"))
    assert torch.equal(r.starts[:-1].long(), starts) and starts[-1] == total
    assert torch.equal(r.order[:total].long(), order[:total] // top) and (r.order[total:-1] == -1).all()
    places = torch.full_like(order, -1)
    places[order[:total]] = torch.arange(total, device="cuda")
    assert torch.equal(r.places[:-1].long(), places)


@pytest.mark.parametrize("n,top,width,t,to,gap", [(3, 70, 2048, 1, 1, 0), (40, 33, 701, 0, 2, 1), (7, 65, 96, 2, 1, 8), (700, 3, 4099, 1, 2, 2), (1, 1, 1, 2, 2, 0), (3, 3, 777, 2, 2, 0), (5, 2, 1000, 1, 2, 8), (64, 8, 128, 0, 1, 0), (200, 5, 333, 1, 0, 3), (300, 2, 4096, 1, 1, 0), (17, 32, 520, 2, 1, 4), (1000, 4, 96, 0, 0, 16)])
def test_combine(lib, n, top, width, t, to, gap):
    import torch
    rng = np.random.default_rng(n + width)
    rows = n * top
    y = torch.full((rows, width + gap), float("nan"), dtype=_dtype(t), device="cuda")
    y[:, :width] = torch.from_numpy(rng.standard_normal((rows, width)) * 4).to(_dtype(t)).cuda()
    places = rng.integers(0, rows, (n, top)).astype(np.int32)     # (one place may be asked for twice)
    places[rng.random(places.shape) < 0.2] = -1
    places[0, 0] = rows - 1
    if n > 2:
        places[1], places[2, 0] = -1, rows                       # nothing at all; beyond the last
        places[2, -1] = -2 ** 31
    gates = rng.random((n, top)).astype(np.float32)
    gates[places < 0] = np.nan                                    # (not looked at)
    out = torch.full((n + 1, width + gap), 7.0, dtype=_dtype(to), device="cuda")
    pd, gd = torch.from_numpy(places).cuda(), torch.from_numpy(gates).cuda()
    assert lib.spgk_combine_rows(y.data_ptr(), t, width + gap, rows, pd.data_ptr(), gd.data_ptr(), n, top, width, out.data_ptr(), to, width + gap, None) == 0, lib.spgk_error_string()
    got = out.double().cpu().numpy()
    assert (got[n] == 7).all() and (got[:, width:] == 7).all()
    yv = y[:, :width].double().cpu().numpy()
    want, size = plain.combine(yv, places, gates), plain.combine(np.abs(yv), places, gates)
    assert (np.abs(got[:n, :width] - want) <= top * 2.0 ** -24 * size + HALF[to] * np.abs(want) * (1 + top * 2.0 ** -20) + (2.0 ** -25 if to == 0 else 0)).all()
    none = torch.full((n + 1, width + gap), 7.0, dtype=_dtype(to), device="cuda")                 # no rows at all
    assert lib.spgk_combine_rows(None, t, width + gap, 0, pd.data_ptr(), gd.data_ptr(), n, top, width, none.data_ptr(), to, width + gap, None) == 0
    assert (none[:n, :width] == 0).all()


@pytest.mark.parametrize("n,experts,top,k,hidden,units,t", [(1, 16, 2, 512, 1024, 300, 1), (1, 3, 3, 129, 70, 33, 0), (37, 5, 2, 300, 500, 200, 1), (300, 8, 2, 512, 640, 384, 1), (64, 100, 4, 256, 384, 128, 0), (2000, 4, 1, 200, 300, 100, 1)])
def test_the_whole_way(spg, lib, n, experts, top, k, hidden, units, t):
    """Router, quantised rows in the experts' order, two layers of experts, sums: each as by its own test, together as a program calls them, eagerly and from a graph."""
    import torch
    rng = np.random.default_rng(n + experts)
    (w1, w1v), (w2, w2v) = _random(spg, experts * hidden, k, rng), _random(spg, experts * units, hidden, rng)
    b1, b2 = (torch.from_numpy(rng.standard_normal(experts * u).astype(np.float32)).cuda() for u in (hidden, units))
    logits = _logits(rng, n, experts, "masked")
    x, l = torch.zeros(n, k, dtype=_dtype(t), device="cuda"), torch.zeros(n, experts, device="cuda")
    r = Route(n, experts, top)
    x8, h8 = Packed(spg, n * top, k), Packed(spg, n * top, hidden)
    z, out = torch.full((n * top, units), float("nan"), dtype=_dtype(t), device="cuda"), torch.full((n, units), 9.0, dtype=_dtype(t), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def way(stream):
        r.run(lib, l, 2, experts, 1, stream)
        assert lib.spgk_fp8_quantize(x.data_ptr(), t, k, n, r.order.data_ptr(), x8.ref, stream) == 0
        assert lib.spgk_experts_fp8(w1.ref, experts, b1.data_ptr(), 3, x8.ref, r.starts.data_ptr(), None, 0, 0, h8.ref, status.data_ptr(), stream) == 0
        assert lib.spgk_experts_fp8(w2.ref, experts, b2.data_ptr(), 6, h8.ref, r.starts.data_ptr(), z.data_ptr(), t, units, None, status.data_ptr(), stream) == 0
        assert lib.spgk_combine_rows(z.data_ptr(), t, units, n * top, r.places.data_ptr(), r.gates.data_ptr(), n, top, units, out.data_ptr(), t, units, stream) == 0

    def check(values, logits):
        torch.cuda.synchronize()
        assert status.item() == 0
        r.check(logits, 1)
        _, gates, starts, order, places = plain.route(logits, top, True)
        total = starts[-1]
        xq = plain.values(*plain.quantize(values[order[:total]]))
        code, scale = h8.host()
        hq = plain.values(code, scale)[:total]                    # (as it came: its own rounding is checked next, the second layer from it)
        zv = np.zeros((n * top, units))
        for e in range(experts):
            rows = slice(starts[e], starts[e + 1])
            if starts[e] == starts[e + 1]:
                continue
            h = plain.ACTS[3](xq[rows] @ w1v[e * hidden:(e + 1) * hidden].T + b1.cpu().numpy()[e * hidden:(e + 1) * hidden])
            most = np.abs(np.pad(h, ((0, 0), (0, -hidden % 128)))).reshape(h.shape[0], -1, 128).max(-1)
            # half a step of the element, or of the grid's finest where that is more; what the fp32 sums may be off by is far below it
            step = np.maximum(np.abs(h) * 2.0 ** -4, np.repeat(most, 128, 1)[:, :hidden] * 2.0 ** -17) + np.abs(xq[rows]) @ np.abs(w1v[e * hidden:(e + 1) * hidden]).T * (k + 33) * 2.0 ** -23
            assert (np.abs(hq[rows] - h) <= step * 1.001).all()
            zv[rows] = hq[rows] @ w2v[e * units:(e + 1) * units].T + b2.cpu().numpy()[e * units:(e + 1) * units]
            size = np.abs(hq[rows]) @ np.abs(w2v[e * units:(e + 1) * units]).T + 4
            got = z.double().cpu().numpy()[rows]
            fine = np.abs(zv[rows]) < 65000
            assert (np.abs(got - zv[rows]) <= size * (hidden + 33) * 2.0 ** -23 + np.abs(zv[rows]) * HALF[t] + 2.0 ** -25)[fine].all()
        got, zg = out.double().cpu().numpy(), z.double().cpu().numpy()
        want, size = plain.combine(zg, places, gates), plain.combine(np.abs(zg), places, gates)
        fine = size < 65000                                       # (some of the fp16 rows are infinite)
        with np.errstate(invalid="ignore"):
            off = np.abs(got - want)
        assert (off <= size * 2.0 ** -16 + HALF[t] * np.abs(want) + 2.0 ** -25)[fine].all()

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    for turn in range(3):
        values = rng.standard_normal((n, k))
        logits = _logits(rng, n, experts, "masked" if turn else "plain")
        x.copy_(torch.from_numpy(values))
        l.copy_(torch.from_numpy(logits))
        torch.cuda.synchronize()
        if turn == 0:
            way(None)
        elif turn == 1:
            with torch.cuda.graph(graph, stream=stream):
                way(torch.cuda.current_stream().cuda_stream)
            graph.replay()
        else:
            graph.replay()
        check(x.double().cpu().numpy(), l.double().cpu().numpy())
