"""What a network has and gives as operands of the kernel-level operators: its weights in microscaled 4 bits, its outputs as rows of logits."""
import numpy as np
import pytest

import mx4_plain as plain
from test_gpu_mx4 import Packed, lib  # noqa: F401  (lib: fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def net(spg):
    net = spg.Network.build([784, 512, 1000], [spg.abi.ACT_RELU, spg.abi.ACT_NONE], spg.abi.WEIGHT_INITIALIZATION_NONE)
    rng = np.random.default_rng(5)
    net.weights[:] = rng.standard_normal(net.weights.size).astype(np.float32) / 16
    net.biases[:] = rng.standard_normal(net.biases.size).astype(np.float32) / 4
    net.sync_weights()
    yield net
    net.free()


def _draws(lib, logits, u, p):
    import torch
    n, width = logits.shape
    held = [torch.full((n,), p, device="cuda"), torch.from_numpy(u).cuda()]
    tokens, kept = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    assert lib.spgk_sample_rows(logits.data_ptr(), 2, width, n, width, None, None, held[0].data_ptr(), None, held[1].data_ptr(), tokens.data_ptr(), None, kept.data_ptr(), None) == 0
    torch.cuda.synchronize()
    rows = logits.double().cpu().numpy()
    want = [plain.sample_row(rows[i], 1.0, None, float(np.float32(p)), None, float(u[i])) for i in range(n)]
    assert tokens.tolist() == [w[0] for w in want] and kept.tolist() == [w[2] for w in want]


def test_tokens_drawn_from_what_a_network_gives(lib, net):
    """forward_batch from device memory to device memory, and a token a row, on one stream."""
    import torch
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.random((70, 784), dtype=np.float32)).cuda()
    logits = torch.empty((70, 1000), device="cuda")
    torch.cuda.synchronize()
    net.forward_batch_ptr(x.data_ptr(), 70, logits.data_ptr())
    net.synchronize()
    w1, w2 = (net.weights[a:b].reshape(s).astype(np.float64) for a, b, s in ((0, 401408, (512, 784)), (401408, 913408, (1000, 512))))
    want = np.maximum(x.double().cpu().numpy() @ w1.T + net.biases[:512], 0) @ w2.T + net.biases[512:]
    assert np.abs(logits.cpu().numpy() - want).max() <= 2e-3 * np.abs(want).max()        # (that these are the logits; how close they are is tested elsewhere)
    _draws(lib, logits, rng.random(70).astype(np.float32), 0.9)


def test_a_networks_weights_in_four_bits(lib, spg, net):
    """Both layers' weights uploaded and quantised, then the forward in 4 bits to tokens, every step against its plain form on what the step before gave."""
    import torch
    rng = np.random.default_rng(7)
    n = 70
    packed, values, start = [], [], 0
    for out, k in ((512, 784), (1000, 512)):
        w = net.weights[start:start + out * k].reshape(out, k)
        start += out * k
        held, m = torch.from_numpy(w.copy()).cuda(), Packed(spg, out, k)
        assert lib.spgk_mx4_quantize(held.data_ptr(), 2, k, m.ref, None) == 0
        torch.cuda.synchronize()
        code, scale = plain.quantize(w.astype(np.float64))
        assert np.array_equal(m.host()[0], code) and np.array_equal(m.host()[1], scale)
        packed.append(m)
        values.append(plain.values(code, scale, k))
    b = torch.from_numpy(net.biases.copy()).cuda()
    x = torch.from_numpy(rng.random((n, 784), dtype=np.float32)).cuda()
    x4, h4, logits = Packed(spg, n, 784), Packed(spg, n, 512), torch.empty((n, 1000), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.spgk_mx4_quantize(x.data_ptr(), 2, 784, x4.ref, None) == 0
    assert lib.spgk_layer_mx4(packed[0].ref, b.data_ptr(), spg.abi.ACT_RELU, x4.ref, None, 0, 0, h4.ref, status.data_ptr(), None) == 0
    assert lib.spgk_layer_mx4(packed[1].ref, b.data_ptr() + 4 * 512, spg.abi.ACT_NONE, h4.ref, logits.data_ptr(), 2, 1000, None, status.data_ptr(), None) == 0
    assert lib.spgk_gemm_tc_status(status.data_ptr(), None) == 0
    # the hidden layer: an element is off by one of its block's units at most (half way between 4 and 6), by two where a value of nearly 8 stays at 6
    xv = plain.values(*plain.quantize(x.double().cpu().numpy()), 784)
    z = np.maximum(xv @ values[0].T + net.biases[:512], 0)
    code, scale = h4.host()
    hv = plain.values(code, scale, 512)
    unit = np.repeat(np.exp2(scale.astype(float) - 127), 32, 1)
    assert (np.abs(hv - z) <= 2 * unit + 1e-6).all()
    want = hv @ values[1].T + net.biases[512:]
    tol = (512 // 64 + 1) * 65 * 2.0 ** -24 * (np.abs(hv) @ np.abs(values[1]).T + np.abs(net.biases[512:]))
    assert (np.abs(logits.double().cpu().numpy() - want) <= tol).all()
    _draws(lib, logits, rng.random(n).astype(np.float32), 0.9)


@pytest.mark.parametrize("n,width", [(150, 16411), (5, 70001), (9, 1000)])
@pytest.mark.parametrize("cuts", ["none", "k", "p", "kpm", "K", "Kp"])
def test_logits_far_from_zero_and_low_temperatures(lib, n, width, cuts):
    """|largest| / temperature beyond the range of the weights from the table: each weight by itself in 64 bits, rows kept and rows read pass by pass."""
    import torch
    from test_gpu_sample_rows import _check, _draw
    rng = np.random.default_rng(n + width + len(cuts))
    x = (rng.standard_normal((n, width)) * 3).astype(np.float32)
    t = rng.uniform(0.4, 1.5, n)
    x[::2] += 6000
    t[1::2] = 2e-3
    x[1::2] += rng.uniform(-5, 30, (len(x[1::2]), 1)).astype(np.float32)
    xd = torch.from_numpy(x).cuda()
    k = rng.integers(300, 900, n) if "K" in cuts else rng.integers(1, 250, n) if "k" in cuts else None
    p = rng.uniform(0.05, 1.02, n) if "p" in cuts else None
    m = rng.uniform(0.0, 0.2, n) if "m" in cuts else None
    u = rng.random(n).astype(np.float32)
    _check(_draw(lib, xd, t, k, p, m, u), xd, t, k, p, m, u)
