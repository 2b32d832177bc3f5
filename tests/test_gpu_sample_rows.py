"""Tokens drawn from rows of logits against a sort and sums in 64 bits."""
import numpy as np
import pytest

import mx4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib(spg, has_gpu):
    assert has_gpu, "no CUDA device"
    return spg.lib()


def _draw(lib, x, t=None, k=None, p=None, m=None, u=None, kind=2, width=None, stream=None):
    """x: device rows (a view keeps its stride); the others host arrays or None"""
    import torch
    n = x.shape[0]
    width = width or x.shape[1]

    def dev(a, dt):
        return None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype=dt)).cuda()
    held = [dev(t, np.float32), dev(k, np.int32), dev(p, np.float32), dev(m, np.float32), dev(u, np.float32)]
    tokens = torch.full((n + 1,), -77, dtype=torch.int32, device="cuda")
    probs = torch.full((n + 1,), -7.0, device="cuda")
    kept = torch.full((n + 1,), -77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc = lib.spgk_sample_rows(x.data_ptr(), kind, x.stride(0), n, width, *[None if h is None else h.data_ptr() for h in held], tokens.data_ptr(), probs.data_ptr(), kept.data_ptr(), stream)
    assert rc == 0, lib.spgk_error_string()
    torch.cuda.synchronize()
    assert tokens[n] == -77 and probs[n] == -7 and kept[n] == -77
    return tokens[:n].cpu().numpy(), probs[:n].double().cpu().numpy(), kept[:n].cpu().numpy()


def _check(got, x, t, k, p, m, u):
    rows = x.double().cpu().numpy()
    for i in range(len(rows)):
        at = [None if a is None else a[i] for a in (k, p, m)]
        want = plain.sample_row(rows[i], 1.0 if t is None else float(np.float32(t[i])), at[0], None if at[1] is None else float(np.float32(at[1])), None if at[2] is None else float(np.float32(at[2])),
                                float(np.float32(u[i])))
        assert (got[0][i], got[2][i]) == (want[0], want[2]), (i, got[0][i], got[1][i], got[2][i], want)
        # a weight is good to 2^-30 of itself and 2^-45 of the largest, and so is their total; then one rounding to 32 bits
        assert abs(got[1][i] - want[1]) <= want[1] * (2.0 ** -24 + 2 * 2.0 ** -30) + 2.0 ** -44, (i, got[1][i], want[1])


SIZES = [(1, 1), (3, 2), (5, 31), (2, 33), (7, 1000), (300, 17), (3, 4097), (2, 32769), (40, 5000), (2, 50001), (1, 131072), (1, 262144), (150, 9001)]
CUTS = ["none", "k", "p", "m", "kp", "km", "pm", "kpm", "greedy"]


@pytest.mark.parametrize("n,width", SIZES)
@pytest.mark.parametrize("cuts", CUTS)
def test_draws(lib, n, width, cuts):
    import torch
    rng = np.random.default_rng(n * 7 + width + len(cuts))
    kind = (n + width + len(cuts)) % 3
    x = torch.from_numpy((rng.standard_normal((n, width + n % 4)) * rng.uniform(0.5, 5)).astype(np.float32)).cuda()
    x = x.to({0: torch.float16, 1: torch.bfloat16, 2: torch.float32}[kind])[:, :width]
    t = np.zeros(n) if cuts == "greedy" else rng.uniform(0.4, 1.5, n)
    k = rng.integers(1, min(width, 300) + 2, n) if "k" in cuts else None
    p = rng.uniform(0.05, 1.02, n) if "p" in cuts else None
    m = rng.uniform(0.0, 0.2, n) if "m" in cuts else None
    u = rng.random(n).astype(np.float32)
    _check(_draw(lib, x, t, k, p, m, u, kind), x, t, k, p, m, u)


def test_a_vocabulary_masked_in_runs(lib):
    """Whole stretches of a long row masked, as the unused end of a vocabulary is: some CTAs of the row have nothing, some a single logit."""
    import torch
    rng = np.random.default_rng(2)
    n, width = 9, 60000
    x = rng.standard_normal((n, width)).astype(np.float32)
    for i in range(n):
        x[i, width * (i + 1) // 10:] = -np.inf
        x[i, -1 - i] = 0.25 * i
        if i % 3 == 2:
            x[i, :5000 * i] = -np.inf
    xd = torch.from_numpy(x).cuda()
    for k, p, m in ((50, None, None), (256, 0.9, None), (3, None, 0.1), (None, 0.6, None), (700, None, None)):
        t, u = np.full(n, 0.9), rng.random(n).astype(np.float32)
        a = [None if v is None else np.full(n, v) for v in (k, p, m)]
        _check(_draw(lib, xd, t, *a, u), xd, t, *a, u)


@pytest.mark.parametrize("width", [40, 3000, 70000])
def test_masks_ties_and_odd_values(lib, width):
    """Rows without a logit, with one, with equal ones only, infinities, NaN, differences beyond the weights' range."""
    import torch
    rng = np.random.default_rng(width)
    x = rng.standard_normal((16, width)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, width // 3] = -5.0
    x[3] = 1.5                                               # all equal
    x[4, ::2] = np.nan
    x[5, 7], x[5, width - 1] = np.inf, np.inf
    x[6] = np.where(rng.random(width) < 0.9, -np.inf, x[6])
    x[7] = np.round(x[7])                                    # few different values
    x[8] *= 1e30
    x[9] = np.where(np.arange(width) % 2, -0.0, 0.0)
    x[10] = -3.4e38
    x[11] = np.float32(-3.4028235e38)
    x[11, 3] = np.float32(3.4028235e38)
    x[12] = 1e-42 * rng.standard_normal(width)
    x[13] = 0.0
    x[13, 5] = np.nextafter(np.float32(0), np.float32(1))
    x[14] = np.linspace(-1, 1, width, dtype=np.float32)
    x[15] = np.inf
    xd = torch.from_numpy(x).cuda()
    for t, k, p, m in ((1.0, None, None, None), (0.8, 5, None, None), (1.0, None, 0.5, None), (1.3, None, None, 0.1), (1.0, 30, 0.7, 0.05), (0.0, None, None, None), (1.0, 7, 0.2, None)):
        u = rng.random(16).astype(np.float32)
        a = [None if v is None else np.full(16, v) for v in (k, p, m)]
        t = np.full(16, t)
        _check(_draw(lib, xd, t, *a, u), xd, t, *a, u)


def test_arguments_at_their_ends(lib):
    """Cuts that do not cut, cuts to one, temperatures and random numbers at and beyond the ends of their ranges."""
    import torch
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((12, 700)).astype(np.float32)).cuda()
    nan, inf = np.nan, np.inf
    u = np.array([0, 1 - 2.0 ** -24, 0.5, 0, 0.3, 0.99, 1 - 2.0 ** -24, 0.2, 0.7, 0.1, 0.5, 0.5])
    t = np.array([1, 1, nan, -1, inf, 1e-3, 100, 1e-38, 1, 1, 1, 1.0])
    _check(_draw(lib, x, t, None, None, None, u), x, t, None, None, None, u)
    one = np.ones(12)
    k = np.array([0, -5, 700, 701, 2 ** 31 - 1, 1, 2, 699, 1, 3, 50, 100])
    _check(_draw(lib, x, one, k, None, None, u), x, one, k, None, None, u)
    p = np.array([0, -1, 1, 2, 1e-30, 0.999999, 0.5, 0.1, 0.9, 1e-3, 0.25, 0.75])
    _check(_draw(lib, x, None, None, p, None, u), x, None, None, p, None, u)
    m = np.array([0, -1, 1, 2, 1e-30, 0.999999, 0.5, 0.1, 0.9, 1e-3, 0.25, 0.75])
    _check(_draw(lib, x, one, k, p, m, u), x, one, k, p, m, u)
    # beyond the ends: a NaN is no cut, random numbers are taken to [0, 1)
    got = _draw(lib, x, one, None, np.full(12, nan), np.full(12, nan), np.array([-1, nan, 1, 2, inf, -inf] * 2))
    assert (got[2] == 700).all() and set(got[0][[0, 1, 5]]) == {0} and set(got[0][[2, 3, 4]]) == {699}


def test_shares_of_many_draws(lib):
    """The same row with evenly spaced numbers: every token as often as its weight says, in the order of the vocabulary."""
    import torch
    n = 4096
    w = np.array([0.1, 0.0, 0.3, 0.05, 0.25, 0.3])
    with np.errstate(divide="ignore"):
        x = torch.from_numpy(np.log(w).astype(np.float32)).cuda().expand(n, 6).contiguous()
    u = (np.arange(n) / n).astype(np.float32)
    tokens = _draw(lib, x, None, None, None, None, u)[0]
    assert (np.diff(tokens) >= 0).all()
    assert (np.abs(np.bincount(tokens, minlength=6) - w * n) <= 1).all()


def test_outputs_that_are_not_wanted_and_replay(lib):
    import torch
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((6, 20000)).astype(np.float32)).cuda()
    u = torch.rand(6, device="cuda")
    p = torch.full((6,), 0.9, device="cuda")
    tokens = torch.full((6,), -9, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def go():
        assert lib.spgk_sample_rows(x.data_ptr(), 2, 20000, 6, 20000, None, None, p.data_ptr(), None, u.data_ptr(), tokens.data_ptr(), None, None, side.cuda_stream) == 0
    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        go()
    for _ in range(3):
        x.normal_()
        u.uniform_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        rows = x.double().cpu().numpy()
        for i in range(6):
            assert tokens[i].item() == plain.sample_row(rows[i], 1.0, None, float(np.float32(0.9)), None, u[i].item())[0]
    del graph


@pytest.mark.parametrize("cuts", ["none", "k", "p", "kpm", "K", "Kp"])
@pytest.mark.parametrize("kind,pad", [(2, 0), (2, 3), (1, 0), (0, 5)])
def test_many_long_rows(lib, cuts, kind, pad):
    """Rows that are read pass by pass, at every alignment of their ends; the first of them masked, equal, or full of ties."""
    import torch
    rng = np.random.default_rng(len(cuts) + 7 * kind + pad)
    n, width = 150, 16411
    x = (rng.standard_normal((n, width + pad)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1] = 0.5
    x[2] = np.round(x[2])
    x[3, ::2] = np.nan
    x[4, 5], x[4, width - 1] = np.inf, np.inf
    x[5, 9000:] = -np.inf
    x = torch.from_numpy(x).cuda().to({0: torch.float16, 1: torch.bfloat16, 2: torch.float32}[kind])[:, :width]
    t = rng.uniform(0.4, 1.5, n)
    t[6] = 0
    k = rng.integers(300, 3000, n) if "K" in cuts else rng.integers(1, 250, n) if "k" in cuts else None
    p = rng.uniform(0.05, 1.02, n) if "p" in cuts else None
    m = rng.uniform(0.0, 0.2, n) if "m" in cuts else None
    u = rng.random(n).astype(np.float32)
    _check(_draw(lib, x, t, k, p, m, u, kind), x, t, k, p, m, u)


@pytest.mark.parametrize("n", [2, 130])
def test_rows_of_one_value_but_few(lib, n):
    """More equal logits in one bin than sums of 32 bits would hold, below a few larger ones: kept in shared memory, and read pass by pass."""
    import torch
    rng = np.random.default_rng(n)
    width = 200001
    x = np.full((n, width), -0.3, np.float32)
    x[:, 77], x[:, 150000] = 1.0, 0.25
    x[0, 5] = 9.0
    x[1, 1000:1100] = rng.standard_normal(100)
    if n > 2:
        x[2:, ::3] += rng.uniform(0, 0.01, (n - 2, 66667)).astype(np.float32)
    xd = torch.from_numpy(x).cuda()
    rows = np.unique(np.r_[0, 1, rng.integers(0, n, 10)])                        # (a plain sort of each)
    for cuts in ((None, 0.5, None), (None, 0.99, None), (1000, 0.7, None), (None, None, None), (70000, None, None), (None, 0.3, 0.2)):
        t, u = np.full(n, 0.7), rng.random(n).astype(np.float32)
        a = [None if v is None else np.full(n, v) for v in cuts]
        got = _draw(lib, xd, t, *a, u)
        _check([g[rows] for g in got], xd[torch.from_numpy(rows).cuda()], t[rows], *[None if v is None else v[rows] for v in a], u[rows])
