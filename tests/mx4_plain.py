"""Plain forms in 64 bits of the operators on microscaled 4-bit numbers and on rows of logits, for their tests."""
import math

import numpy as np

SIZES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
ACTS = {0: lambda v: 1 / (1 + np.exp(-v)), 1: lambda v: np.where(v > 0, v, 0), 2: np.tanh, 3: lambda v: np.where(v > 0, v, 0.01 * v),
        4: lambda v: np.where(v > 1, 1 + 0.01 * (v - 1), np.where(v < 0, 0.01 * v, v)), 5: lambda v: v, 6: lambda v: v}


def scale_place(cols, row, block):
    tiles = -(-cols // 128)
    return (row // 128 * tiles + block // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + block % 4


def quantize(x):
    """(codes [rows][blocks * 32], scale bytes [rows][blocks]) of rows of finite or other values."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(-1)
    a = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    e = np.full(a.shape, -127)
    some = a > 0
    e[some] = np.maximum(np.frexp(a[some])[1] - 1 - 2, -127)
    unit = np.exp2(e.astype(float))[..., None]
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.minimum(np.abs(np.where(bad[..., None], 0, v)) / unit, 6.0)
    code = np.zeros(v.shape, np.uint8)
    for i in range(1, 8):
        half = (SIZES[i - 1] + SIZES[i]) / 2
        code += (q > half) | ((q == half) & (i % 2 == 0))
    code = np.where(bad[..., None], 0, code | (np.signbit(v).astype(np.uint8) << 3)).astype(np.uint8)
    return code.reshape(rows, blocks * 32), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale, cols):
    size = SIZES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(float) - 127))
    return (size.reshape(scale.shape + (32,)) * s[..., None]).reshape(code.shape)[:, :cols]


def pack(code, scale, cols, pitch=None):
    """codes bytes [rows][pitch] and the scales in tiles"""
    rows = code.shape[0]
    need = scale.shape[1] * 16
    out = np.zeros((rows, pitch or need), np.uint8)
    out[:, :need] = code[:, 0::2] | code[:, 1::2] << 4
    tiles = np.zeros(-(-rows // 128) * -(-cols // 128) * 512, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(scale.shape[1]), indexing="ij")
    tiles[scale_place(cols, r, b)] = scale
    return out, tiles


def unpack(codes, tiles, rows, cols):
    blocks = -(-cols // 32)
    c = codes[:rows, :blocks * 16]
    code = np.stack((c & 15, c >> 4), -1).reshape(rows, blocks * 32)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    return code, tiles[scale_place(cols, r, b)]


def sample_row(l, t, k, p, m, u):
    """(token, probability, how many were left) of one row in 64 bits; None for a cut that is not asked for"""
    l = np.where(np.isnan(l), -np.inf, l.astype(float))
    first = int(np.argmax(l))
    top = l[first]
    if top == -np.inf:
        return -1, 0.0, 0
    if not t > 0:
        return first, 1.0, 1
    order = np.argsort(-l, kind="stable")[:int((l > -np.inf).sum())]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l[order] == top, 1.0, 0.0 if np.isinf(top) else np.exp((l[order] - top) / t))
    count = len(order) if k is None or k < 1 else min(len(order), int(k))
    total = math.fsum(w[:count])
    cuts = [count]
    if p is not None and p < 1:
        cuts.append(int(np.searchsorted(np.cumsum(w[:count]), p * total)) + 1)
    if m is not None and m > 0:
        cuts.append(int((w >= m).sum()))
    count = max(1, min(cuts))
    by_index = np.argsort(order[:count])
    w, order = w[:count][by_index], order[:count][by_index]
    sums = np.cumsum(w)
    u = u if u > 0 else 0.0
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), int(np.flatnonzero(w)[-1]))
    return int(order[at]), w[at] / sums[-1], count
