"""Routes of more pairs than one cluster has, which go in parts whose counts lie in the results' memory on the way: every type, both kinds of gates, padded rows, closed experts."""
import numpy as np
import pytest

from test_gpu_fp8 import _dtype, lib  # noqa: F401  (lib: fixture)
from test_gpu_route import Route

pytestmark = pytest.mark.gpu


def _plain(logits, top, normalise):
    """(chosen, gates, starts, order, places) in 64 bits, by sorts of all there is"""
    import torch
    l = torch.where(logits.isnan(), float("-inf"), logits.double()) + 0.0
    n, experts = l.shape
    value, index = torch.sort(l, dim=1, descending=True, stable=True)
    open_ = value[:, :top] > float("-inf")
    chosen = torch.where(open_, index[:, :top], -1)
    m = value[:, :1]
    w = torch.where(l == m, 1.0, torch.where(m.isinf(), 0.0, torch.exp(l - torch.where(m.isinf(), 0.0, m))))
    mine = torch.where(open_, torch.gather(w, 1, index[:, :top]), 0.0)
    total = mine.sum(1, keepdim=True) if normalise else w.sum(1, keepdim=True)
    gates = torch.where(open_, mine / total, 0.0)
    flat = torch.where(open_, chosen, experts).view(-1)
    by = torch.sort(flat, stable=True)[1]
    count = int(open_.sum())
    starts = torch.searchsorted(flat[by], torch.arange(experts + 1, device="cuda"))
    order = torch.full_like(by, -1)
    order[:count] = by[:count] // top
    places = torch.full_like(by, -1)
    places[by[:count]] = torch.arange(count, device="cuda")
    return chosen.view(-1), gates.view(-1), starts, order, places


def _logits(n, experts, kind, t):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(n + experts)
    l = torch.randn(n, experts, device="cuda", generator=g) * 3

    def some(share):
        return torch.rand(l.shape, device="cuda", generator=g) < share
    if kind == "ties":
        l = torch.round(l)
        l[some(0.1)] = -0.0
    if kind != "plain":
        l[some(0.3)] = float("-inf")
        l[some(0.05)] = float("nan")
        l[::97] = float("-inf")                                   # nothing at all
        l[1::97, 1:] = float("nan")                               # one at most
        l[2::97] = torch.where(some(0.1)[2::97], float("inf"), l[2::97])
        l[3::97, experts // 2] = float("inf")
    return l.to(_dtype(t))


# (the last part has the rest: 63 rows of parts of 32, 63 of 32, 43 of 22, 1385 of 1000, one row more than a whole number of parts, and 79 of 64)
SHAPES = [(16415, 256, 8), (607, 1024, 32), (5477, 5, 3), (16385, 1000, 1), (20001, 64, 2), (20047, 3, 1)]


@pytest.mark.parametrize("n,experts,top", SHAPES)
@pytest.mark.parametrize("t,pad", [(0, 0), (0, 3), (1, 0), (1, 8), (2, 0), (2, 1)])
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_routes_in_parts(lib, kind, t, pad, n, experts, top):
    import torch
    assert n * top > 16384
    full = torch.full((n, experts + pad), 1e4, dtype=_dtype(t), device="cuda")               # what is beside a row is not read
    full[:, :experts] = _logits(n, experts, kind, t)
    logits = full[:, :experts]
    far = min(2 * float(torch.nan_to_num(logits.double(), 0.0, 0.0, 0.0).abs().max()), 104.0)
    for normalise in (0, 1):
        r = Route(n, experts, top)
        r.run(lib, full, t, experts + pad, normalise)
        want = _plain(logits, top, normalise)
        got = (r.chosen, r.gates, r.starts, r.order, r.places)
        assert all(v[-1].item() == -77 for v in got)             # (what lies behind the results)
        for i in (0, 2, 3, 4):
            assert torch.equal(got[i][:-1].long(), want[i]), ("chosen", "", "starts", "order", "places")[i]
        # as derived in test_gpu_route: the difference's rounding, 2 ulp of expf, the additions, the division
        tol = (2 * (far + 4) + 40) * 2.0 ** -24 * want[1] + 2.0 ** -126
        assert ((got[1][:-1].double() - want[1]).abs() <= tol).all()
        assert (got[1][:-1][want[0] < 0] == 0).all()


def test_routes_in_parts_again_and_from_a_graph(lib):
    """The counts of a call before lie in the results' memory when the next begins: the same memory, other logits, eagerly and replayed."""
    import torch
    n, experts, top = 16415, 256, 8
    r, x = Route(n, experts, top), torch.zeros((n, experts), dtype=torch.bfloat16, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    for turn, kind in enumerate(("masked", "plain", "ties", "masked")):
        x.copy_(_logits(n, experts, kind, 1).roll(turn, 0))
        torch.cuda.synchronize()
        if turn < 2:
            r.run(lib, x, 1, experts, 0)
        else:
            if turn == 2:
                with torch.cuda.graph(graph, stream=stream):
                    r.run(lib, x, 1, experts, 0, torch.cuda.current_stream().cuda_stream)
            graph.replay()
        torch.cuda.synchronize()
        want = _plain(x, top, 0)
        for got, expect in zip((r.chosen, r.starts, r.order, r.places), (want[0], *want[2:])):
            assert torch.equal(got[:-1].long(), expect)
