"""The operators on microscaled 4-bit numbers and on rows of logits, as measurable cases.

`quantize`: rows of values to blocks of 4-bit elements with a scale each, and back to the values they stand for.
`layer`: a dense layer on two such matrices, with bias and activation.
`mlp`: rows quantised, a hidden layer whose output stays in 4 bits, and the layer behind it.
`sample`: a token drawn from every row of logits, with temperature, top-k, top-p and min-p, from given random numbers.

`listed()` names the cases to watch, `draw(rng)` gives others of the same ranges, `prepare` makes what a program has in hand
(packed weights, activations, random numbers, buffers that it keeps), `run` is one pass: the operators written out in elementary
torch operations, or, with `own` set, the library's calls.  `exact` says in 64 bits, by other means, what a pass has to give.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"f16": 0, "bf16": 1, "f32": 2}                       # SPGK_T_*
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
ACTS = {"sigmoid": 0, "relu": 1, "tanh": 2, "leaky": 3, "foo52": 4, "none": 6}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)             # half way between neighbours


def listed():
    return [
        # one sample's activations before a layer: latency
        {"name": "quantize_1x8192_bf16", "kind": "quantize", "rows": 1, "cols": 8192, "pad": 0, "type": "bf16", "out": "bf16"},
        # a batch of odd width out of a wider buffer
        {"name": "quantize_3001x777_f16", "kind": "quantize", "rows": 3001, "cols": 777, "pad": 24, "type": "f16", "out": "f32"},
        # a layer's weights, or the activations of a large batch: bandwidth
        {"name": "quantize_16384x8192_f32", "kind": "quantize", "rows": 16384, "cols": 8192, "pad": 0, "type": "f32", "out": "f32"},
        # the first layer of the large net for one sample: the weights are read once
        {"name": "layer_1x8192x16384_f32", "kind": "layer", "rows": 1, "in": 8192, "units": 16384, "act": "foo52", "out": "f32"},
        # its second layer for a small served batch
        {"name": "layer_64x16384x16384_bf16", "kind": "layer", "rows": 64, "in": 16384, "units": 16384, "act": "foo52", "out": "bf16"},
        # a ragged layer and a batch that ends in a part of a tile
        {"name": "layer_3001x777x333_f16", "kind": "layer", "rows": 3001, "in": 777, "units": 333, "act": "tanh", "out": "f16"},
        # a layer of the wide net on its batch: products
        {"name": "layer_16384x8192x8192_bf16", "kind": "layer", "rows": 16384, "in": 8192, "units": 8192, "act": "leaky", "out": "bf16"},
        # eight served samples through a hidden layer to logits
        {"name": "mlp_8x8192x16384x1000_f16", "kind": "mlp", "rows": 8, "in": 8192, "hidden": 16384, "units": 1000, "act": "foo52", "type": "f32", "out": "f16"},
        # a batch through two layers of the wide net
        {"name": "mlp_2048x4096x8192x4096_bf16", "kind": "mlp", "rows": 2048, "in": 4096, "hidden": 8192, "units": 4096, "act": "leaky", "type": "bf16", "out": "bf16"},
        # one answer out of the nets' thousand classes: latency
        {"name": "sample_1x1000_f32", "kind": "sample", "rows": 1, "width": 1000, "pad": 0, "type": "f32", "temperature": 0.7, "top_k": 40, "top_p": 0.95, "min_p": 0.0, "masked": 0.0},
        # a served batch with every cut, part of the vocabulary masked, logits with many ties
        {"name": "sample_64x50001_bf16", "kind": "sample", "rows": 64, "width": 50001, "pad": 7, "type": "bf16", "temperature": 0.9, "top_k": 50, "top_p": 0.9, "min_p": 0.02, "masked": 0.3},
        # a large batch over a long vocabulary, cut by mass alone: bandwidth
        {"name": "sample_256x131072_f32", "kind": "sample", "rows": 256, "width": 131072, "pad": 0, "type": "f32", "temperature": 0.8, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "masked": 0.0},
    ]


def _size(rng, most, least=1):
    """A whole number, its logarithm spread evenly; one in three a multiple of 32."""
    v = int(round(math.exp(rng.uniform(math.log(least), math.log(most + 0.49)))))
    v = max(32, v // 32 * 32) if rng.random() < 0.33 and most >= 32 else v
    return max(least, min(most, v))


def draw(rng):
    kind = rng.choice(("quantize", "layer", "layer", "mlp", "sample", "sample"))
    if kind == "quantize":
        cols = _size(rng, 16384)
        return {"kind": kind, "rows": _size(rng, min(16384, (1 << 26) // cols)), "cols": cols, "pad": rng.choice((0, 0, 1, 8, 24)), "type": rng.choice(("f32", "f16", "bf16")),
                "out": rng.choice(("f32", "bf16"))}
    if kind == "layer":
        k, units = _size(rng, 16384), _size(rng, 16384)
        return {"kind": kind, "rows": _size(rng, max(1, min(16384, (1 << 26) // units, (1 << 39) // (k * units)))), "in": k, "units": units, "act": rng.choice(tuple(ACTS)),
                "out": rng.choice(("f32", "f16", "bf16"))}
    if kind == "mlp":
        k, hidden, units = _size(rng, 8192, 16), _size(rng, 16384, 16), _size(rng, 4096)
        return {"kind": kind, "rows": _size(rng, max(1, min(4096, (1 << 37) // (hidden * (k + units))))), "in": k, "hidden": hidden, "units": units, "act": rng.choice(("relu", "leaky", "foo52")),
                "type": rng.choice(("f32", "f16", "bf16")), "out": rng.choice(("f16", "bf16"))}
    width = _size(rng, 200003)
    return {"kind": kind, "rows": _size(rng, min(512, max(1, (1 << 24) // width))), "width": width, "pad": rng.choice((0, 0, 1, 8)), "type": rng.choice(("f32", "f16", "bf16")),
            "temperature": rng.choice((0.0, round(rng.uniform(0.3, 1.6), 3), round(rng.uniform(0.3, 1.6), 3))), "top_k": rng.choice((0, _size(rng, 2000))),
            "top_p": rng.choice((1.0, round(rng.uniform(0.1, 0.99), 3))), "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.2), 4))), "masked": rng.choice((0.0, round(rng.uniform(0.0, 0.9), 2)))}


def work(case):
    rows = case["rows"]
    if case["kind"] == "quantize":
        n = rows * case["cols"]
        packed = rows * (-(-case["cols"] // 32)) * 17
        return {"bytes": n * (BYTES[case["type"]] + BYTES[case["out"]]) + 2 * packed, "flops": 2 * n}
    if case["kind"] == "layer":
        blocks = -(-case["in"] // 32)
        return {"bytes": (rows + case["units"]) * blocks * 17 + 4 * case["units"] + rows * case["units"] * BYTES[case["out"]], "flops": 2 * rows * case["in"] * case["units"]}
    if case["kind"] == "mlp":
        k, hidden, units = case["in"], case["hidden"], case["units"]
        weights = 17 * (hidden * (-(-k // 32)) + units * (-(-hidden // 32))) + 4 * (hidden + units)
        return {"bytes": rows * k * BYTES[case["type"]] + weights + rows * units * BYTES[case["out"]], "flops": 2 * rows * hidden * (k + units)}
    n = rows * case["width"]
    return {"bytes": n * BYTES[case["type"]] + 28 * rows, "flops": 8 * n}


# ---- the packed form --------------------------------------------------------------------------------------------------------

def _pitch(cols):
    return -(-cols // 32) * 16


def _tiles(scales):
    """Scale bytes [rows][blocks] in tiles of 128 rows x 4 blocks: byte (row % 32) * 16 + row % 128 / 32 * 4 + block % 4 of a tile."""
    rows, blocks = scales.shape
    r, b = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros(r * 128, b * 4, dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(r, 4, 32, b, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _untiled(tiles, rows, blocks):
    r, b = -(-rows // 128), -(-blocks // 4)
    return tiles.view(r, b, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, b * 4)[:rows, :blocks]


def _encode(x):
    """Rows of values to (codes [rows][blocks * 32] as numbers 0..15, scale bytes [rows][blocks])."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, 32)
    a = v.abs().amax(-1)
    fine = torch.isfinite(v).all(-1)
    a = torch.where(fine, a, torch.ones_like(a))
    e = torch.where(a > 0, torch.frexp(a)[1] - 3, torch.full_like(a, -127, dtype=torch.int32)).clamp(-127, 127)
    # the scale is a power of two and |v| / scale below 8: exact in 64 bits
    q = (v.abs() * torch.exp2(-e.double()).unsqueeze(-1)).nan_to_num(0.0, 0.0, 0.0)
    code = torch.zeros_like(v, dtype=torch.uint8)
    for i, border in enumerate(BORDERS):
        code += (q > border) if i % 2 == 0 else (q >= border)     # half way: to the even code
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    code = torch.where(fine.unsqueeze(-1), code, torch.zeros_like(code))
    scale = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code.view(rows, blocks * 32), scale


def _decode(code, scale, cols):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=code.device)
    s = torch.exp2(scale.double() - 127).float()
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    rows, blocks = scale.shape
    return (table[code.long()].view(rows, blocks, 32) * s.unsqueeze(-1)).view(rows, blocks * 32)[:, :cols]


def _pack(x):
    """A packed matrix as a program holds it."""
    code, scale = _encode(x)
    return {"codes": (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), "scales": _tiles(scale), "rows": x.shape[0], "cols": x.shape[1]}


def _room(rows, cols):
    b = -(-cols // 32)
    return {"codes": torch.empty(rows, b * 16, dtype=torch.uint8, device="cuda"),
            "scales": torch.empty(-(-rows // 128) * (-(-b // 4)) * 512, dtype=torch.uint8, device="cuda"), "rows": rows, "cols": cols}


def _values(m):
    c = m["codes"]
    code = torch.stack((c & 15, c >> 4), -1).view(m["rows"], -1)
    return _decode(code, _untiled(m["scales"], m["rows"], -(-m["cols"] // 32)), m["cols"])


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _activations(rows, cols, g):
    """Values whose columns differ in size, as a layer's outputs do."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    return x * torch.exp2(torch.randn(1, cols, device="cuda", generator=g))


def _weights(units, k, g):
    return _pack(torch.randn(units, k, device="cuda", generator=g) / math.sqrt(k)), torch.randn(units, device="cuda", generator=g) * 0.1


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = case["rows"]
    s = {"case": case}
    if case["kind"] == "quantize":
        cols = case["cols"]
        full = _activations(rows, cols + case["pad"], g).to(TYPES[case["type"]])
        s["x"] = full[:, :cols]
        s["packed"] = _room(rows, cols)
        s["y"] = torch.empty(rows, cols, dtype=TYPES[case["out"]], device="cuda")
    elif case["kind"] == "layer":
        s["w"], s["bias"] = _weights(case["units"], case["in"], g)
        s["x"] = _pack(_activations(rows, case["in"], g))
        s["y"] = torch.empty(rows, case["units"], dtype=TYPES[case["out"]], device="cuda")
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    elif case["kind"] == "mlp":
        s["w1"], s["bias1"] = _weights(case["hidden"], case["in"], g)
        s["w2"], s["bias2"] = _weights(case["units"], case["hidden"], g)
        s["x"] = _activations(rows, case["in"], g).to(TYPES[case["type"]])
        s["x4"], s["h4"] = _room(rows, case["in"]), _room(rows, case["hidden"])
        s["y"] = torch.empty(rows, case["units"], dtype=TYPES[case["out"]], device="cuda")
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        width = case["width"]
        full = torch.randn(rows, width + case["pad"], device="cuda", generator=g) * 2.5
        if case["masked"]:
            hidden = torch.rand(rows, width + case["pad"], device="cuda", generator=g) < case["masked"]
            if rows >= 8:
                hidden[rows // 3] = True                                    # a row that allows nothing
            full = full.masked_fill(hidden, float("-inf"))
        s["x"] = full.to(TYPES[case["type"]])[:, :width]

        def each(v):
            return v * (0.8 + 0.2 * torch.rand(rows, device="cuda", generator=g))
        s["temperature"] = each(case["temperature"])
        s["top_k"] = torch.ceil(each(case["top_k"])).to(torch.int32) if case["top_k"] else None
        s["top_p"] = each(case["top_p"]) if case["top_p"] < 1 else None
        s["min_p"] = each(case["min_p"]) if case["min_p"] else None
        s["u"] = torch.rand(rows, device="cuda", generator=g)
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["probs"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        s["kept"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "leaky":
        return torch.where(v > 0, v, 0.01 * v)
    if act == "foo52":
        return torch.where(v > 1, 1 + 0.01 * (v - 1), torch.where(v < 0, 0.01 * v, v))
    if act == "tanh":
        return torch.tanh(v)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    return v


def _dense(x, w, bias, act):
    return _act(x @ w.t() + bias, act)


def _sample(x, temperature, top_k, top_p, min_p, u):
    """Weights and their sums in 64 bits: the last bits decide on which side of a border a number falls."""
    rows, width = x.shape
    l = x.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l)
    top = l.amax(1, keepdim=True)
    t = temperature.double().unsqueeze(1)
    greedy = ~(t > 0)
    w = torch.exp((l - top) / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(l == top, torch.ones_like(w), w)
    w = torch.where(torch.isinf(l) & (l < 0), torch.zeros_like(w), w)
    ls, order = torch.sort(l, dim=1, descending=True, stable=True)
    ws = torch.gather(w, 1, order)
    rank = torch.arange(width, device=x.device).unsqueeze(0)
    keep = ls > -math.inf
    if top_k is not None:
        k = top_k.long().unsqueeze(1)
        keep = keep & ((rank < k) | (k < 1))
    ws = torch.where(keep, ws, torch.zeros_like(ws))
    if top_p is not None:
        p = top_p.double().unsqueeze(1)
        upto = ws.cumsum(1)
        keep = keep & ((upto - ws < p * upto[:, -1:]) | (p >= 1))
    if min_p is not None:
        m = min_p.double().unsqueeze(1)
        keep = keep & ((ws >= m) | (m <= 0))
    keep = torch.where(greedy, rank < 1, keep | (rank < 1)) & (ls > -math.inf)
    left = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, torch.zeros_like(ws)))
    upto = left.cumsum(1)
    total = upto[:, -1]
    goal = (u.double() * total).unsqueeze(1)
    token = ((upto <= goal).sum(1)).clamp(max=width - 1)
    none = total == 0
    prob = left.gather(1, token.unsqueeze(1)).squeeze(1) / torch.where(none, torch.ones_like(total), total)
    return {"tokens": torch.where(none, torch.full_like(token, -1), token).to(torch.int32), "probs": prob.float(), "kept": keep.sum(1).to(torch.int32)}


def _plain(s):
    case = s["case"]
    if case["kind"] == "quantize":
        code, scale = _encode(s["x"].float())
        return _decode(code, scale, case["cols"]).to(TYPES[case["out"]])
    if case["kind"] == "layer":
        return _dense(_values(s["x"]), _values(s["w"]), s["bias"], case["act"]).to(TYPES[case["out"]])
    if case["kind"] == "mlp":
        # the hidden layer in 64 bits: its values are rounded to few of them, and some lie next to a border
        x = _decode(*_encode(s["x"].float()), case["in"])
        h = _dense(x.double(), _values(s["w1"]).double(), s["bias1"].double(), case["act"])
        h = _decode(*_encode(h), case["hidden"])
        return _dense(h, _values(s["w2"]), s["bias2"], "none").to(TYPES[case["out"]])
    return _sample(s["x"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["u"])


def _handles(s):
    """The library and what its calls take, made once as a program would."""
    import ctypes
    import spingalett_b200 as spg

    lib = spg.lib()

    def matrix(m):
        return ctypes.byref(spg.abi.Mx4(m["codes"].data_ptr(), m["scales"].data_ptr(), m["rows"], m["cols"], m["codes"].shape[1]))

    def at(t):
        return None if t is None else t.data_ptr()

    case = s["case"]
    calls = []
    if case["kind"] == "quantize":
        packed = matrix(s["packed"])
        calls += [(lib.spgk_mx4_quantize, (at(s["x"]), CODES[case["type"]], s["x"].stride(0), packed)),
                  (lib.spgk_mx4_dequantize, (packed, at(s["y"]), CODES[case["out"]], case["cols"]))]
    elif case["kind"] == "layer":
        calls += [(lib.spgk_layer_mx4, (matrix(s["w"]), at(s["bias"]), ACTS[case["act"]], matrix(s["x"]), at(s["y"]), CODES[case["out"]], case["units"], None, at(s["status"])))]
    elif case["kind"] == "mlp":
        x4, h4 = matrix(s["x4"]), matrix(s["h4"])
        calls += [(lib.spgk_mx4_quantize, (at(s["x"]), CODES[case["type"]], case["in"], x4)),
                  (lib.spgk_layer_mx4, (matrix(s["w1"]), at(s["bias1"]), ACTS[case["act"]], x4, None, 0, 0, h4, at(s["status"]))),
                  (lib.spgk_layer_mx4, (matrix(s["w2"]), at(s["bias2"]), ACTS["none"], h4, at(s["y"]), CODES[case["out"]], case["units"], None, at(s["status"])))]
    else:
        calls += [(lib.spgk_sample_rows, (at(s["x"]), CODES[case["type"]], s["x"].stride(0), case["rows"], case["width"], at(s["temperature"]), at(s["top_k"]), at(s["top_p"]),
                                          at(s["min_p"]), at(s["u"]), at(s["tokens"]), at(s["probs"]), at(s["kept"])))]
    return lib, calls


def _library(s):
    if "calls" not in s:
        s["calls"] = _handles(s)
    lib, calls = s["calls"]
    stream = torch.cuda.current_stream().cuda_stream
    for call, args in calls:
        if call(*args, stream) != 0:
            raise RuntimeError(lib.spgk_error_string().decode())
    if s["case"]["kind"] == "sample":
        return {"tokens": s["tokens"], "probs": s["probs"], "kept": s["kept"]}
    return s["y"]


def run(s):
    return _library(s) if own else _plain(s)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------------

def _exact_values(m):
    """A packed matrix read element by element from the description of its layout."""
    rows, cols = m["rows"], m["cols"]
    blocks = -(-cols // 32)
    c = torch.arange(cols, device="cuda")
    byte = m["codes"][:, c // 2].long() >> (4 * (c % 2))
    size = torch.where(byte & 6 == 0, 0.5 * (byte & 1), torch.exp2(((byte >> 1) & 3).double() - 1) * (1 + 0.5 * (byte & 1)))
    r, b = torch.arange(rows, device="cuda").unsqueeze(1), (c // 32).unsqueeze(0)
    place = ((r // 128) * (-(-blocks // 4)) + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4
    e = m["scales"][place].double()
    return torch.where(byte & 8 != 0, -size, size) * torch.where(e == 255, torch.full_like(e, math.nan), torch.exp2(e - 127))


def _exact_rounding(x):
    """Every value of x rounded to its block's grid: the nearest of the eight sizes, of two equally near ones that with the even code."""
    rows, cols = x.shape
    pad = -cols % 32
    v = torch.nn.functional.pad(x.double(), (0, pad)).view(-1, 32)
    sizes = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    out = torch.empty_like(v)
    for i in range(0, v.shape[0], 1 << 18):
        p = v[i:i + (1 << 18)]
        a = p.abs().amax(1, keepdim=True)
        bad = ~torch.isfinite(p).all(1, keepdim=True)
        unit = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -125))).clamp(min=-125) - 2)
        unit = torch.where(a >= 8 * unit, 2 * unit, torch.where(a < 4 * unit, unit / 2, unit)).clamp(min=2.0 ** -127)
        far = (p.abs().unsqueeze(-1) / unit.unsqueeze(-1) - sizes).abs()
        near = far.amin(-1, keepdim=True)
        hit = far == near
        odd = torch.arange(8, device=x.device) % 2 == 1
        hit = hit & ~(odd & (hit.sum(-1, keepdim=True) > 1))
        got = torch.copysign(sizes[hit.to(torch.uint8).argmax(-1)], p) * unit
        out[i:i + (1 << 18)] = torch.where(bad, torch.full_like(got, math.nan), got)
    return out.view(rows, cols + pad)[:, :cols]


def _exact_act(v, act):
    f = {"relu": lambda: v.clamp(min=0), "leaky": lambda: torch.maximum(v, 0.01 * v), "tanh": lambda: torch.tanh(v), "sigmoid": lambda: torch.sigmoid(v), "none": lambda: v,
         "foo52": lambda: v.clamp(0, 1) + 0.01 * (v - v.clamp(0, 1))}
    return f[act]()


def _exact_dense(x, w, bias, act):
    return _exact_act(torch.addmm(bias.double(), x, w.T), act)


def _exact_row(l, t, k, p, m, u):
    """One row: its order by sorting, its cuts by counting along it."""
    l = np.where(np.isnan(l), -np.inf, l)
    first = int(np.argmax(l))
    top = l[first]
    if top == -np.inf:
        return -1, 0.0, 0
    if not t > 0:
        return first, 1.0, 1
    order = np.argsort(-l, kind="stable")[: int(np.count_nonzero(l > -np.inf))]
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / t))
    count = len(order) if k is None or k < 1 else min(len(order), int(k))
    total = math.fsum(w[:count]) if count < 5000 else float(np.sum(w[:count]))
    cuts = [count]
    if p is not None and p < 1:
        cuts.append(int(np.searchsorted(np.cumsum(w[:count]), p * total)) + 1)
    if m is not None and m > 0:
        cuts.append(int(np.count_nonzero(w >= m)))
    count = max(1, min(cuts))
    index = np.argsort(order[:count])
    w, order = w[:count][index], order[:count][index]
    sums = np.cumsum(w)
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), count - 1)
    return int(order[at]), w[at] / sums[-1], count


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_rounding(s["x"])
    if case["kind"] == "layer":
        return _exact_dense(_exact_values(s["x"]), _exact_values(s["w"]), s["bias"], case["act"])
    if case["kind"] == "mlp":
        h = _exact_dense(_exact_rounding(s["x"]), _exact_values(s["w1"]), s["bias1"], case["act"])
        return _exact_dense(_exact_rounding(h), _exact_values(s["w2"]), s["bias2"], "none")
    x = s["x"].double().cpu().numpy()

    def column(name):
        return [None] * case["rows"] if s[name] is None else s[name].double().cpu().tolist()
    got = [_exact_row(*row) for row in zip(x, column("temperature"), column("top_k"), column("top_p"), column("min_p"), column("u"))]
    return {"tokens": torch.tensor([g[0] for g in got], dtype=torch.int32), "probs": torch.tensor([g[1] for g in got], dtype=torch.float64),
            "kept": torch.tensor([g[2] for g in got], dtype=torch.int32)}
