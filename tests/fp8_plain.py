"""Plain forms in 64 bits of the operators on 8-bit numbers with a scale for each block of 128, and of routing rows to experts and back, for their tests."""
import numpy as np

from mx4_plain import ACTS  # noqa: F401

BLOCK = 128
_code = np.arange(128)
SIZES = np.where(_code < 8, _code * 2.0 ** -9, (8 + _code % 8) * np.exp2(_code // 8 - 10.0))      # what codes 0 to 126 stand for
SIZES[127] = np.nan


def blocks(cols):
    return -(-cols // BLOCK)


def scale_place(rows, row, block):
    return (block // 4 * rows + row) * 4 + block % 4


def quantize(x):
    """(codes [rows][cols], scale bytes [rows][blocks]) of rows of finite or other values."""
    rows, cols = x.shape
    v = np.zeros((rows, blocks(cols) * BLOCK))
    v[:, :cols] = x
    v = v.reshape(rows, blocks(cols), BLOCK)
    bad = ~np.isfinite(v).all(-1)
    a = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    e = np.full(a.shape, -127)
    for k in range(-127, 128):                                  # the least power of two by which it comes to 448 or less
        e = np.where(a > 448.0 * 2.0 ** k, k + 1, e)
    q = np.abs(np.where(bad[..., None], 0, v)) / np.exp2(e.astype(float))[..., None]
    near = np.searchsorted(SIZES[:127], q)                      # the first that is not below
    near = np.minimum(near, 126)
    low = np.maximum(near - 1, 0)
    up, down = SIZES[near] - q, q - SIZES[low]
    code = np.where((up < down) | ((up == down) & (near % 2 == 0)), near, low).astype(np.uint8)
    code = np.where(bad[..., None], 0, code | (np.signbit(v).astype(np.uint8) << 7)).astype(np.uint8)
    return code.reshape(rows, blocks(cols) * BLOCK)[:, :cols], np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale):
    """What codes [rows][cols] with scale bytes [rows][blocks] stand for."""
    size = SIZES[code & 127] * np.where(code & 128, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(float) - 127))
    return size * np.repeat(s, BLOCK, 1)[:, :code.shape[1]]


def pack(code, scale, pitch, fill=0xA5):
    """Code bytes [rows][pitch] and the scales in their order; `fill` in what is not looked at"""
    rows, cols = code.shape
    out = np.full((rows, pitch), fill, np.uint8)
    out[:, :cols] = code
    words = np.full(-(-blocks(cols) // 4) * rows * 4, fill, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(scale.shape[1]), indexing="ij")
    words[scale_place(rows, r, b)] = scale
    return out, words


def unpack(codes, words, rows, cols):
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks(cols)), indexing="ij")
    return codes[:rows, :cols], words[scale_place(rows, r, b)]


def ranges(starts, rows):
    """The groups' rows out of starts of any kind: none below zero, an earlier one or beyond the last row"""
    out, last = [], 0
    for e in range(len(starts) - 1):
        lo = max(last, min(max(int(starts[e]), 0), rows))
        hi = max(lo, min(max(int(starts[e + 1]), 0), rows))
        out.append((lo, hi))
        last = hi
    return out


def route(logits, top, normalise):
    """(chosen, gates, starts, order, places) of rows of logits."""
    l = np.where(np.isnan(logits), -np.inf, logits.astype(float)) + 0.0
    rows, experts = l.shape
    chosen, gates = np.full((rows, top), -1), np.zeros((rows, top))
    for n in range(rows):
        by = np.lexsort((np.arange(experts), -l[n]))[:top]
        by = by[l[n][by] > -np.inf]
        if len(by) == 0:
            continue
        m = l[n].max()
        with np.errstate(invalid="ignore"):
            w = np.where(l[n] == m, 1.0, np.exp(l[n] - m) if np.isfinite(m) else 0.0)
        chosen[n, :len(by)] = by
        gates[n, :len(by)] = w[by] / (w[by].sum() if normalise else w.sum())
    places, order, starts = np.full((rows, top), -1), [], [0]
    for e in range(experts):
        for n, j in zip(*np.nonzero(chosen == e)):
            places[n, j] = len(order)
            order.append(n)
        starts.append(len(order))
    return chosen, gates, np.array(starts), np.array(order + [-1] * (rows * top - len(order)), int), places


def combine(y, places, gates):
    out = np.zeros((places.shape[0], y.shape[1]))
    for n in range(places.shape[0]):
        for p, g in zip(places[n], gates[n]):
            if 0 <= p < y.shape[0]:
                with np.errstate(invalid="ignore"):
                    out[n] += float(g) * y[p]
    return out
