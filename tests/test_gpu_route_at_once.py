"""Rows to experts and back on several streams at a time: routes of all three ways, quantising by their order, layers of experts and sums, each stream with results of its own."""
import numpy as np
import pytest

from test_gpu_fp8 import Packed, _random, lib  # noqa: F401  (lib: fixture)
from test_gpu_route import Route
from test_gpu_route_parts import _logits, _plain

pytestmark = pytest.mark.gpu

# (rows, experts, top_k, inputs, units): one block of threads, one cluster, parts
WAYS = [(9, 16, 2, 384, 200), (700, 40, 4, 256, 130), (3000, 64, 8, 128, 72)]


class Way:
    """A layer of experts around which rows are routed; its operands are shared by all streams, its results are not."""

    def __init__(self, spg, lib, n, experts, top, k, units):
        import torch
        rng = np.random.default_rng(n)
        self.spg, self.lib, self.n, self.experts, self.top, self.k, self.units = spg, lib, n, experts, top, k, units
        self.logits = _logits(n, experts, "ties", 1)
        self.x = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32)).cuda()
        self.w = _random(spg, experts * units, k, rng)[0]

    def results(self):
        import torch
        return (Route(self.n, self.experts, self.top), Packed(self.spg, self.n * self.top, self.k), torch.full((self.n * self.top, self.units), 5.0, device="cuda"),
                torch.full((self.n, self.units), 5.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))

    def run(self, results, stream):
        r, x8, y, out, status = results
        pairs = self.n * self.top
        r.run(self.lib, self.logits, 1, self.experts, 0, stream)
        assert self.lib.spgk_fp8_quantize(self.x.data_ptr(), 2, self.k, self.n, r.order.data_ptr(), x8.ref, stream) == 0
        assert self.lib.spgk_experts_fp8(self.w.ref, self.experts, None, 1, x8.ref, r.starts.data_ptr(), y.data_ptr(), 2, self.units, None, status.data_ptr(), stream) == 0
        assert self.lib.spgk_combine_rows(y.data_ptr(), 2, self.units, pairs, r.places.data_ptr(), r.gates.data_ptr(), self.n, self.top, self.units, out.data_ptr(), 2, self.units, stream) == 0


def _same(a, b):
    import torch
    tensors = [(getattr(a[0], name), getattr(b[0], name)) for name in ("chosen", "gates", "starts", "order", "places")]
    tensors += [(a[1].codes, b[1].codes), (a[1].words, b[1].words), (a[2], b[2]), (a[3], b[3])]
    return all(torch.equal(s.nan_to_num(9.0) if s.is_floating_point() else s, t.nan_to_num(9.0) if t.is_floating_point() else t) for s, t in tensors)


@pytest.mark.parametrize("replayed", [False, True])
def test_ways_at_once(spg, lib, replayed):
    """Four streams go through all ways in orders of their own, six times, without a wait; what each leaves is, bit for bit, what a way alone leaves, whose route is checked against sorts."""
    import torch
    ways = [Way(spg, lib, *w) for w in WAYS]
    alone = []
    for way in ways:
        alone.append(way.results())
        way.run(alone[-1], None)
        torch.cuda.synchronize()
        want = _plain(way.logits, way.top, 0)
        for got, expect in zip((alone[-1][0].chosen, alone[-1][0].starts, alone[-1][0].order, alone[-1][0].places), (want[0], *want[2:])):
            assert torch.equal(got[:-1].long(), expect)
    streams = [torch.cuda.Stream() for _ in range(4)]
    results = [[way.results() for way in ways] for _ in streams]

    def through(i, stream):
        for turn in range(6):
            for j in range(len(ways)):
                k = (i + j * (1 + i % 2) + turn) % len(ways)
                ways[k].run(results[i][k], stream)
    torch.cuda.synchronize()
    if replayed:
        graphs = []
        for i, stream in enumerate(streams):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                through(i, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for _ in range(2):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
    else:
        for i, stream in enumerate(streams):
            through(i, stream.cuda_stream)
    torch.cuda.synchronize()
    for mine in results:
        for way, got, want in zip(ways, mine, alone):
            assert got[4].item() == 0 and _same(got, want), (way.n, way.experts)
